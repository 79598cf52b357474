// Norms before and after a sub-layer, fused with its gate and residual scale, for packed batches (gfx950).
//
//   p = Norm_post(hidden) * post_weight                        (fp32)
//   r = bf16(alpha * residual + gate[q] * p)                   the carried residual, written
//   y = bf16(Norm_pre(r) * mul[q] + add[q])                    written as it is, as MX or as ROW codes
//
// for every row of a packed [T, H] batch, q the row's request: gate, mul and add are one row of H
// for all requests or one per request. A row whose id names no request is not computed: it is left as it
// was, or written as zeros where the caller has just allocated the outputs.
//
// The sum r is the only value between the input and y that is rounded (it is an output, and the norm that
// follows in the block reads it again). Row statistics are fp32: mean and variance in two passes over
// the registers, so no difference of large sums is taken; the root is fp64.
//
// One wavefront owns a row: lane l holds columns 512 c + 8 l .. + 7 of chunk c, as in the adaLN pass.
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
  int64_t T;
  int H, nch;
  int post_norm, norm, quant;
  int zero_rest;
  uint16_t* residual_out;
  void* out;
  uint8_t* scales;
};

namespace {

constexpr int kRsrcWord3 = 0x00020000;
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, kRsrcWord3);
}

__device__ __forceinline__ void load8f(__amdgpu_buffer_rsrc_t r, int lane, int c, float (&v)[8]) {
  const u32x4 v0 = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 32, c * 2048, 0);
  const u32x4 v1 = __builtin_amdgcn_raw_buffer_load_b128(r, lane * 32 + 16, c * 2048, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = __uint_as_float(v0[j]);
    v[4 + j] = __uint_as_float(v1[j]);
  }
}

// Mean and 1 / sqrt(variance or mean square + eps) of a row held as packed bf16 pairs; columns past H are zero.
template <int NCH>
__device__ __forceinline__ void row_stats(const uint32_t (&xp)[NCH][4], int norm, int lane, int H, float eps, float& mu,
                                          float& rs) {
  mu = 0.0f;
  rs = 1.0f;
  if (norm == WANMI_NORM_NONE) return;
  if (norm == WANMI_NORM_LAYER) {
    float s1 = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) s1 += bf16_lo(xp[c][j]) + bf16_hi(xp[c][j]);
    mu = wave_sum_f32_asc(s1) / (float)H;
  }
  float s2 = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const bool ok = c * 512 + lane * 8 < H;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d0 = bf16_lo(xp[c][j]) - mu, d1 = bf16_hi(xp[c][j]) - mu;
      s2 += ok ? d0 * d0 + d1 * d1 : 0.0f;
    }
  }
  s2 = wave_sum_f32_asc(s2);
  rs = (float)(1.0 / sqrt((double)(s2 / (float)H) + (double)eps));
}

template <int NCH>
__global__ __launch_bounds__(256) void adaln_sandwich_kernel(SandwichArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = a.H;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.T) return;
  const int id = a.ids ? __builtin_amdgcn_readfirstlane(a.ids[row]) : 0;
  const bool live = (uint32_t)id < (uint32_t)a.requests;
  if (!live && !a.zero_rest) return;

  const __amdgpu_buffer_rsrc_t r_ro = rsrc(a.residual_out + row * H, 2 * (int64_t)H);
  const int64_t out_bytes = a.quant == WANMI_QUANT_NONE ? 2 * (int64_t)H : a.quant == WANMI_QUANT_MX ? (int64_t)H : (int64_t)H + 4;
  uint8_t* out_row = reinterpret_cast<uint8_t*>(a.out) + row * out_bytes;
  const __amdgpu_buffer_rsrc_t r_o = rsrc(out_row, out_bytes);
  const __amdgpu_buffer_rsrc_t r_s = rsrc(a.quant == WANMI_QUANT_MX ? a.scales + row * (int64_t)(H / 32) : nullptr,
                                          a.quant == WANMI_QUANT_MX ? H / 32 : 0);
  if (!live) {
    const u32x4 z = {0u, 0u, 0u, 0u};
    for (int c = 0; c < a.nch; ++c) {
      store_b128_guarded(z, r_ro, lane * 16, c * 1024);
      if (a.quant == WANMI_QUANT_NONE) {
        store_b128_guarded(z, r_o, lane * 16, c * 1024);
      } else {
        // (the packed row ends in the 4 bytes of its scale: written below)
        if (c * 512 + lane * 8 < H) __builtin_amdgcn_raw_buffer_store_b64(u32x2{0u, 0u}, r_o, lane * 8, c * 512, 0);
        if (a.quant == WANMI_QUANT_MX)
          __builtin_amdgcn_raw_buffer_store_b8((uint8_t)0, r_s, (lane & 3) == 0 ? c * 16 + (lane >> 2) : H, 0, 0);
      }
    }
    if (a.quant == WANMI_QUANT_ROW && lane == 0) __builtin_amdgcn_raw_buffer_store_b32(0u, r_o, H, 0, 0);
    return;
  }

  uint32_t xp[NCH][4], rp[NCH][4];
  const __amdgpu_buffer_rsrc_t r_x = rsrc(a.hidden + row * a.ld_h, 2 * (int64_t)H);
  const __amdgpu_buffer_rsrc_t r_r = rsrc(a.residual + row * a.ld_r, 2 * (int64_t)H);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    // columns past H in the last chunk lie past the descriptors' extents and read as zero
    u32x4 hv = {0u, 0u, 0u, 0u}, rv = {0u, 0u, 0u, 0u};
    if (c < a.nch) {
      hv = __builtin_amdgcn_raw_buffer_load_b128(r_x, lane * 16, c * 1024, 0);
      rv = __builtin_amdgcn_raw_buffer_load_b128(r_r, lane * 16, c * 1024, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) xp[c][j] = hv[j], rp[c][j] = rv[j];
  }
  float mu, rs;
  row_stats<NCH>(xp, a.post_norm, lane, H, a.eps, mu, rs);

  const __amdgpu_buffer_rsrc_t r_w = rsrc(a.post_weight, a.post_weight ? 4 * (int64_t)H : 0);
  const __amdgpu_buffer_rsrc_t r_g = rsrc(a.gate ? a.gate + id * a.ld_gate : nullptr, a.gate ? 4 * (int64_t)H : 0);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (c < a.nch) {
      float wv[8], gv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) wv[j] = gv[j] = 1.0f;
      if (a.post_weight) load8f(r_w, lane, c, wv);
      if (a.gate) load8f(r_g, lane, c, gv);
      u32x4 ov;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = (bf16_lo(xp[c][j]) - mu) * rs * wv[2 * j], p1 = (bf16_hi(xp[c][j]) - mu) * rs * wv[2 * j + 1];
        ov[j] = pack_bf16x2(a.alpha * bf16_lo(rp[c][j]) + gv[2 * j] * p0, a.alpha * bf16_hi(rp[c][j]) + gv[2 * j + 1] * p1);
        if (c * 512 + lane * 8 >= H) ov[j] = 0u;
        xp[c][j] = ov[j];
      }
      store_b128_guarded(ov, r_ro, lane * 16, c * 1024);
    }
  }
  row_stats<NCH>(xp, a.norm, lane, H, a.eps, mu, rs);

  const __amdgpu_buffer_rsrc_t r_m = rsrc(a.mul ? a.mul + id * a.ld_mul : nullptr, a.mul ? 4 * (int64_t)H : 0);
  const __amdgpu_buffer_rsrc_t r_a = rsrc(a.add ? a.add + id * a.ld_add : nullptr, a.add ? 4 * (int64_t)H : 0);
  float amax = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (c < a.nch) {
      const bool ok = c * 512 + lane * 8 < H;
      float mv[8], av[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) mv[j] = 1.0f, av[j] = 0.0f;
      if (a.mul) load8f(r_m, lane, c, mv);
      if (a.add) load8f(r_a, lane, c, av);
      uint32_t yp[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = (bf16_lo(xp[c][j]) - mu) * rs * mv[2 * j] + av[2 * j];
        const float y1 = (bf16_hi(xp[c][j]) - mu) * rs * mv[2 * j + 1] + av[2 * j + 1];
        yp[j] = ok ? pack_bf16x2(y0, y1) : 0u;
      }
      if (a.quant == WANMI_QUANT_NONE) {
        store_b128_guarded(u32x4{yp[0], yp[1], yp[2], yp[3]}, r_o, lane * 16, c * 1024);
      } else if (a.quant == WANMI_QUANT_MX) {
        // a block of 32 columns is 4 consecutive lanes; its exponent is that of its largest |y|
        u16x2 mag = {0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, yp[j] & 0x7FFF7FFFu));
        int e = (int)(max(mag[0], mag[1]) >> 7);
        e = max(e, dpp_i32<0xB1>(e));
        e = max(e, dpp_i32<0x4E>(e));
        const int sexp = max(e - 7, 0);
        const float f = mx_inv_scale(sexp);
        u32x2 cv;
        cv[0] = cvt_e4m3x4(bf16_lo(yp[0]) * f, bf16_hi(yp[0]) * f, bf16_lo(yp[1]) * f, bf16_hi(yp[1]) * f);
        cv[1] = cvt_e4m3x4(bf16_lo(yp[2]) * f, bf16_hi(yp[2]) * f, bf16_lo(yp[3]) * f, bf16_hi(yp[3]) * f);
        __builtin_amdgcn_raw_buffer_store_b64(cv, r_o, lane * 8, c * 512, 0);
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)sexp, r_s, ok && (lane & 3) == 0 ? c * 16 + (lane >> 2) : H, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(yp[j])), fabsf(bf16_hi(yp[j]))));
          xp[c][j] = yp[j];
        }
      }
    }
  }
  if (a.quant == WANMI_QUANT_ROW) {
    amax = wave_max_f32_asc(amax);
    const float dq = fmaxf(amax / 448.0f, 1e-6f);
    const __amdgpu_buffer_rsrc_t r_c = rsrc(out_row, (int64_t)H);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (c < a.nch) {
        float q[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[2 * j] = fminf(fmaxf(bf16_lo(xp[c][j]) / dq, -448.0f), 448.0f);
          q[2 * j + 1] = fminf(fmaxf(bf16_hi(xp[c][j]) / dq, -448.0f), 448.0f);
        }
        u32x2 cv;
        cv[0] = cvt_e4m3x4(q[0], q[1], q[2], q[3]);
        cv[1] = cvt_e4m3x4(q[4], q[5], q[6], q[7]);
        __builtin_amdgcn_raw_buffer_store_b64(cv, r_c, lane * 8, c * 512, 0);
      }
    }
    if (lane == 0) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(dq), r_o, H, 0, 0);
  }
}

template <int NCH>
void launch_sandwich(const SandwichArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((adaln_sandwich_kernel<NCH>), dim3((unsigned)((a.T + 3) / 4)), dim3(256), 0, s, a);
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
  WANMI_REQUIRE(T >= 0 && T < (1LL << 32), WANMI_ERR_ARG, "wanmi_adaln_sandwich: T=%lld must be in [0, 2^32)", (long long)T);
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
  WANMI_REQUIRE(hidden && residual && residual_out && out, WANMI_ERR_ARG,
                "wanmi_adaln_sandwich: hidden, residual, residual_out and out must not be null");
  WANMI_REQUIRE(quant_type != WANMI_QUANT_MX || scales, WANMI_ERR_ARG, "wanmi_adaln_sandwich: MX output needs scales");
  for (int64_t ld : {ld_hidden, ld_residual})
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
  a.nch = (int)((H + 511) / 512);
  a.post_norm = post_norm;
  a.norm = norm_type;
  a.quant = quant_type;
  a.zero_rest = zero_rest;
  a.residual_out = static_cast<uint16_t*>(residual_out);
  a.out = out;
  a.scales = scales;
  hipStream_t s = (hipStream_t)stream;
  if (a.nch <= 2) launch_sandwich<2>(a, s);
  else if (a.nch <= 4) launch_sandwich<4>(a, s);
  else if (a.nch <= 10) launch_sandwich<10>(a, s);
  else if (a.nch <= 20) launch_sandwich<20>(a, s);
  else launch_sandwich<32>(a, s);
  return check_launch("wanmi_adaln_sandwich");
}
