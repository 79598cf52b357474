// Q/K norm and rotary positions on several axes, given per token, for packed batches (gfx950).
//
//   x^ = x * g,  g = gamma / sqrt(mean(x^2) + eps) over each head, over all heads of the row, or g = 1
//   pair (a, b) of channels, i its index in the head, on axis A(i):
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position[row][A(i)] * freq[i]
//
// The pairs are the channels (2i, 2i+1) or (i, i + rot/2) of the head's first `rot` channels; the rest of
// the head keeps x^. All of it in fp32 from one read of x, one rounding to bf16 at the write. Optionally the
// largest norm over each request's rows of every key head, the bound that the constant-max attention needs.
//
// The angle is formed as turns in fp64 (position x freq / 2 pi), reduced to a quarter turn around zero
// and only then rounded, so that it is as exact for a far position as for a near one: sine and cosine
// of at most pi/4 by their power series, whose next terms are below 2e-9 and 3e-8.
//
// One wavefront owns a row of Q or of K. A lane holds units of 16 channels (8 pairs): interleaved pairs
// lie in 32 consecutive bytes, halves in 16 bytes at i and 16 at i + rot/2. A head has D / 16 = 2 .. 16 units, a
// power of two, so a lane's units have the same place u in every head it serves: its 8 angles are read once
// per row. The row's angles are computed once, one pair per lane, and passed through LDS.
#include "wanmi_common.h"

namespace wanmi {
namespace {

constexpr int kMaxPairs = 128;

struct QKAxesArgs {
  struct Part {
    const uint16_t* x;
    int64_t ts, hs;  // elements between rows and between heads
    uint16_t* out;
    int64_t out_ts, out_hs;
    const float* gamma;
    int heads;
  } part[2];
  int64_t T;
  int unit_shift;  // log2 of the units per head
  int rot_units;   // units of a head that turn
  int half;        // rot / 2 (halves)
  int pairs;       // rot / 2
  const void* pos;
  int axes, pos_float;
  const int32_t* ids;
  int requests;
  int norm, zero_rest;
  float eps;
  float* kmax;
  double turns[kMaxPairs];  // freq / 2 pi of every pair
  uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ void sincos_turns(double turns, float& sn, float& cs) {
  const double r = turns - rint(turns);              // [-1/2, 1/2] turns
  const double q = rint(4.0 * r);                    // the nearest quarter: -2 .. 2
  const float t = (float)((r - 0.25 * q) * 6.283185307179586476925);  // [-pi/4, pi/4]
  const float t2 = t * t;
  const float s = t + t * t2 * (-1.0f / 6 + t2 * (1.0f / 120 + t2 * (-1.0f / 5040 + t2 * (1.0f / 362880))));
  const float c = 1.0f + t2 * (-0.5f + t2 * (1.0f / 24 + t2 * (-1.0f / 720 + t2 * (1.0f / 40320))));
  const int k = (int)q & 3;
  const float a = (k & 1) ? c : s, b = (k & 1) ? s : c;
  sn = (k & 2) ? -a : a;
  cs = (k == 1 || k == 2) ? -b : b;
}

// Sum over the 2^shift lanes of a head (aligned groups).
__device__ __forceinline__ float head_sum(float v, int shift) {
  if (shift > 0) v += dpp_f32<0xB1>(v);
  if (shift > 1) v += dpp_f32<0x4E>(v);
  if (shift > 2) v += dpp_f32<0x141>(v);
  if (shift > 3) v += dpp_f32<0x140>(v);
  return v;
}

// NU: units per lane at most (heads * D / 16 / 64, rounded up).
template <int NU, bool kHalves>
__global__ __launch_bounds__(256) void qk_axes_kernel(QKAxesArgs a) {
  __shared__ float tab[4][2][kMaxPairs];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.T) return;
  const QKAxesArgs::Part p = a.part[blockIdx.y];
  const int id = a.ids ? __builtin_amdgcn_readfirstlane(a.ids[row]) : 0;
  const bool live = (uint32_t)id < (uint32_t)a.requests;
  if (!live && !a.zero_rest) return;
  const int u = lane & ((1 << a.unit_shift) - 1);
  const int heads_step = 64 >> a.unit_shift;
  const int h0 = lane >> a.unit_shift;
  const bool turn = u < a.rot_units;
  // the unit's two runs of 8 channels
  const int c0 = kHalves && turn ? 8 * u : 16 * u;
  const int c1 = kHalves && turn ? a.half + 8 * u : 16 * u + 8;
  uint16_t* po = p.out + row * p.out_ts;
  if (!live) {
    const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int h = h0 + i * heads_step;
      if (h < p.heads) {
        store_b128_guarded(z, po + h * p.out_hs + c0);
        store_b128_guarded(z, po + h * p.out_hs + c1);
      }
    }
    return;
  }
  const uint16_t* px = p.x + row * p.ts;
  u32x4 x0[NU], x1[NU];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int h = h0 + i * heads_step;
    x0[i] = x1[i] = u32x4{0u, 0u, 0u, 0u};
    if (h < p.heads) {
      x0[i] = *reinterpret_cast<const u32x4*>(px + h * p.hs + c0);
      x1[i] = *reinterpret_cast<const u32x4*>(px + h * p.hs + c1);
    }
  }
  float* tc = tab[wave][0];
  float* tsn = tab[wave][1];
  for (int i = lane; i < a.pairs; i += 64) {
    const int64_t at = row * a.axes + a.axis[i];
    const double pos = a.pos_float ? (double)reinterpret_cast<const float*>(a.pos)[at]
                                   : (double)reinterpret_cast<const int32_t*>(a.pos)[at];
    float sn, cs;
    sincos_turns(pos * a.turns[i], sn, cs);
    tc[i] = cs;
    tsn[i] = sn;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
  __builtin_amdgcn_wave_barrier();
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    cs[j] = turn ? tc[8 * u + j] : 1.0f;
    sn[j] = turn ? tsn[8 * u + j] : 0.0f;
  }
  float rs = 1.0f;
  if (a.norm == WANMI_QKNORM_ACROSS_HEADS) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ss += bf16_lo(x0[i][j]) * bf16_lo(x0[i][j]) + bf16_hi(x0[i][j]) * bf16_hi(x0[i][j]);
        ss += bf16_lo(x1[i][j]) * bf16_lo(x1[i][j]) + bf16_hi(x1[i][j]) * bf16_hi(x1[i][j]);
      }
    ss = wave_sum_f32_asc(ss);
    rs = (float)(1.0 / sqrt((double)(ss / (float)(p.heads << (a.unit_shift + 4))) + (double)a.eps));
  }
  const int D = 16 << a.unit_shift;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int h = h0 + i * heads_step;
    const bool ok = h < p.heads;
    // the unit's values in memory order: v0 of its first run, v1 of its second
    float v0[8], v1[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v0[2 * j] = bf16_lo(x0[i][j]);
      v0[2 * j + 1] = bf16_hi(x0[i][j]);
      v1[2 * j] = bf16_lo(x1[i][j]);
      v1[2 * j + 1] = bf16_hi(x1[i][j]);
    }
    if (a.norm != WANMI_QKNORM_NONE) {
      float g = rs;
      if (a.norm == WANMI_QKNORM_PER_HEAD) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += v0[j] * v0[j] + v1[j] * v1[j];
        ss = head_sum(ss, a.unit_shift);
        g = (float)(1.0 / sqrt((double)(ss / (float)D) + (double)a.eps));
      }
      if (p.gamma && ok) {
        const float* pg = p.gamma + (a.norm == WANMI_QKNORM_PER_HEAD ? 0 : h * D);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v0[j] *= g * pg[c0 + j];
          v1[j] *= g * pg[c1 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v0[j] *= g, v1[j] *= g;
      }
    }
    if (turn) {
      if (kHalves) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = v0[j], y = v1[j];
          v0[j] = x * cs[j] - y * sn[j];
          v1[j] = x * sn[j] + y * cs[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = v0[2 * j], y = v0[2 * j + 1], z = v1[2 * j], w = v1[2 * j + 1];
          v0[2 * j] = x * cs[j] - y * sn[j];
          v0[2 * j + 1] = x * sn[j] + y * cs[j];
          v1[2 * j] = z * cs[4 + j] - w * sn[4 + j];
          v1[2 * j + 1] = z * sn[4 + j] + w * cs[4 + j];
        }
      }
    }
    if (a.kmax && blockIdx.y == 1) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v0[j] * v0[j] + v1[j] * v1[j];
      ss = head_sum(ss, a.unit_shift);
      // a rounding to bf16 adds at most 2^-8 of a value: the written row's norm is below this
      const float n = sqrtf(ss) * 1.00390625f;
      if (ok && u == 0) atomicMax(reinterpret_cast<unsigned int*>(a.kmax) + (int64_t)id * p.heads + h, __float_as_uint(n));
    }
    if (ok) {
      u32x4 o0, o1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o0[j] = pack_bf16x2(v0[2 * j], v0[2 * j + 1]);
        o1[j] = pack_bf16x2(v1[2 * j], v1[2 * j + 1]);
      }
      store_b128_guarded(o0, po + h * p.out_hs + c0);
      store_b128_guarded(o1, po + h * p.out_hs + c1);
    }
  }
}

__global__ __launch_bounds__(256) void qk_axes_zero_kernel(float* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0.0f;
}

template <int NU>
void launch_qk_axes(const QKAxesArgs& a, bool halves, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + 3) / 4), a.part[1].heads ? 2u : 1u);
  if (halves) hipLaunchKernelGGL((qk_axes_kernel<NU, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((qk_axes_kernel<NU, false>), grid, dim3(256), 0, s, a);
}

}  // namespace
}  // namespace wanmi

extern "C" int wanmi_qk_norm_rope_axes(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
                                       const float* q_gamma, void* q_out, int64_t q_out_token_stride,
                                       int64_t q_out_head_stride, const void* k, int64_t k_token_stride,
                                       int64_t k_head_stride, int k_heads, const float* k_gamma, void* k_out,
                                       int64_t k_out_token_stride, int64_t k_out_head_stride, int64_t T, int head_dim,
                                       const void* positions, int positions_float, int axes, const int* axis_dims,
                                       const double* freqs, int rope_pairs, int norm, float eps,
                                       const int32_t* request_ids, int64_t requests, int zero_rest, float* k_maxnorm,
                                       void* stream) {
  using namespace wanmi;
  clear_error();
  const char* const f = "wanmi_qk_norm_rope_axes";
  WANMI_REQUIRE(T >= 0 && T < (1LL << 32), WANMI_ERR_ARG, "%s: T=%lld must be in [0, 2^32)", f, (long long)T);
  WANMI_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256, WANMI_ERR_UNSUPPORTED,
                "%s: head_dim=%d must be 32, 64, 128 or 256", f, head_dim);
  WANMI_REQUIRE(rope_pairs == WANMI_ROTATE_INTERLEAVED || rope_pairs == WANMI_ROTATE_HALVES, WANMI_ERR_ARG,
                "%s: unknown rope_pairs %d", f, rope_pairs);
  WANMI_REQUIRE(norm == WANMI_QKNORM_NONE || norm == WANMI_QKNORM_PER_HEAD || norm == WANMI_QKNORM_ACROSS_HEADS,
                WANMI_ERR_ARG, "%s: unknown norm %d", f, norm);
  WANMI_REQUIRE(eps >= 0.0f, WANMI_ERR_ARG, "%s: eps must be >= 0", f);
  WANMI_REQUIRE(axes >= 1 && axes <= 8 && axis_dims && freqs, WANMI_ERR_ARG, "%s: 1 to 8 axes with their widths and frequencies", f);
  WANMI_REQUIRE(requests >= 0 && requests < (1LL << 31), WANMI_ERR_ARG, "%s: requests=%lld out of range", f, (long long)requests);
  WANMI_REQUIRE(request_ids || requests >= 1 || T == 0, WANMI_ERR_ARG, "%s: no request to give the rows to", f);
  QKAxesArgs a;
  int rot = 0;
  for (int i = 0; i < axes; ++i) {
    WANMI_REQUIRE(axis_dims[i] >= 0 && axis_dims[i] % 2 == 0 && axis_dims[i] <= head_dim - rot, WANMI_ERR_ARG,
                  "%s: the axes' widths must be even and fit head_dim=%d", f, head_dim);
    for (int j = 0; j < axis_dims[i] / 2; ++j) a.axis[rot / 2 + j] = (uint8_t)i;
    rot += axis_dims[i];
  }
  WANMI_REQUIRE(rot % 16 == 0, WANMI_ERR_UNSUPPORTED, "%s: %d rotary channels: a multiple of 16 is served", f, rot);
  for (int i = 0; i < rot / 2; ++i) a.turns[i] = freqs[i] * 0.15915494309189533577;  // 1 / 2 pi
  WANMI_REQUIRE(q_heads >= 1 && k_heads >= 0, WANMI_ERR_ARG, "%s: q needs heads", f);
  WANMI_REQUIRE(!k_maxnorm || (k_heads >= 1 && requests >= 1), WANMI_ERR_ARG, "%s: k_maxnorm needs k and requests", f);
  const int most = 16384;
  WANMI_REQUIRE((int64_t)q_heads * head_dim <= most && (int64_t)k_heads * head_dim <= most, WANMI_ERR_UNSUPPORTED,
                "%s: heads * head_dim exceeds %d", f, most);
  hipStream_t s = (hipStream_t)stream;
  if (k_maxnorm) {
    const int64_t n = requests * k_heads;
    hipLaunchKernelGGL(qk_axes_zero_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, k_maxnorm, n);
    const int st = check_launch(f);
    if (st != WANMI_OK) return st;
  }
  if (T == 0) return WANMI_OK;
  WANMI_REQUIRE(q && positions && q_out && (!k_heads || (k && k_out)), WANMI_ERR_ARG, "%s: null pointer", f);
  const int64_t strides[8] = {q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride,
                              k_heads ? k_token_stride : 0, k_heads ? k_head_stride : 0, k_heads ? k_out_token_stride : 0,
                              k_heads ? k_out_head_stride : 0};
  for (int64_t v : strides)
    WANMI_REQUIRE(v >= 0 && v % 8 == 0, WANMI_ERR_ARG, "%s: strides must be multiples of 8 elements, got %lld", f, (long long)v);
  for (const void* p : {q, (const void*)q_out, k, (const void*)k_out})
    WANMI_REQUIRE(((uintptr_t)p % 16) == 0, WANMI_ERR_ARG, "%s: tensors must be 16-byte aligned", f);
  a.part[0] = {static_cast<const uint16_t*>(q), q_token_stride, q_head_stride, static_cast<uint16_t*>(q_out),
               q_out_token_stride, q_out_head_stride, q_gamma, q_heads};
  a.part[1] = {static_cast<const uint16_t*>(k), k_token_stride, k_head_stride, static_cast<uint16_t*>(k_out),
               k_out_token_stride, k_out_head_stride, k_gamma, k_heads};
  a.T = T;
  a.unit_shift = head_dim == 32 ? 1 : head_dim == 64 ? 2 : head_dim == 128 ? 3 : 4;
  a.rot_units = rot / 16;
  a.half = a.pairs = rot / 2;
  a.pos = positions;
  a.axes = axes;
  a.pos_float = positions_float;
  a.ids = request_ids;
  a.requests = (int)requests;
  a.norm = norm;
  a.zero_rest = zero_rest;
  a.eps = eps;
  a.kmax = k_maxnorm;
  const int units = (k_heads > q_heads ? k_heads : q_heads) * (head_dim / 16);
  const int nu = (units + 63) / 64;
  const bool halves = rope_pairs == WANMI_ROTATE_HALVES;
  if (nu <= 1) launch_qk_axes<1>(a, halves, s);
  else if (nu <= 2) launch_qk_axes<2>(a, halves, s);
  else if (nu <= 5) launch_qk_axes<5>(a, halves, s);
  else if (nu <= 8) launch_qk_axes<8>(a, halves, s);
  else launch_qk_axes<16>(a, halves, s);
  return check_launch(f);
}
