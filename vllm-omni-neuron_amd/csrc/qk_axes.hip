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
// One wavefront owns a row of Q or of K, and a workgroup of eight rows shares the weight of the norm across heads in LDS (fp32,
// it is as many bytes as the row is read and written). 32760 rows of 40 + 40 heads of 128: 258 us, 5.2 of the 5.5 TB/s
// of a large copy; with the weight from L2 for every row 283. A wave takes one row and ends: the loads of a next one would stand behind the stores of this one in
// the order that a wave waits for them.
//
// A lane holds runs of 8 channels (16 bytes), neighbouring lanes neighbouring runs, so that every instruction moves whole
// lines. Interleaved pairs lie within a run; a run of 64 x i + lane has the same place in its head for every i, since a
// head has D / 8 = 4 .. 32 runs, so its 4 angles are the lane's own. For halves a lane holds the two runs whose
// channels pair up (8 angles), and the same holds for these units of 16 channels. The row's angles are computed
// once, one pair a lane, and passed through LDS.
//
// The largest norm of a request's K rows: the workgroup's largest is compared with what is there already and
// exchanged only if it is larger, since atomics on these few addresses are served one after another for all the
// XCDs (a maximum does not depend on their order). In place, 40 + 40 heads, 3 requests, us without / with the bound (and the
// small launch that clears it): 16 rows 6.9 / 13.6, 1560 15.9 / 20.9, 7800 68 / 77, 32760 270 / 274. With four rows a
// workgroup 7800 rows took 15 us longer.
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

// Sum over the 2^shift lanes of a head (aligned groups, at most 32).
__device__ __forceinline__ float head_sum(float v, int shift) {
  if (shift > 0) v += dpp_f32<0xB1>(v);
  if (shift > 1) v += dpp_f32<0x4E>(v);
  if (shift > 2) v += dpp_f32<0x141>(v);
  if (shift > 3) v += dpp_f32<0x140>(v);
  if (shift > 4) v = add_lane_xor16(v);
  return v;
}

__device__ __forceinline__ void raise_max(float* at, float n) {
  unsigned int* p = reinterpret_cast<unsigned int*>(at);
  const unsigned int bits = __float_as_uint(n);  // (not negative: the order of the bits is the order of the values, NaN on top)
  if (bits > __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(p, bits);
}

// NU: units of 16 channels per lane, heads * D / 16 / 64 rounded up; kWhole: every lane has all of them. kAlone: the
// rows share neither a weight nor maxima.
template <int NU, bool kHalves, bool kWhole, bool kAlone>
__global__ __launch_bounds__(kAlone ? 256 : 512) __attribute__((amdgpu_waves_per_eu(kAlone ? (NU == 2 && kHalves && kWhole ? 5 : 6) : NU <= 3 || (NU <= 5 && (kWhole || !kHalves)) ? 4 : 2))) void qk_axes_kernel(QKAxesArgs a) {
  extern __shared__ __attribute__((aligned(1024))) float gam[];  // [run slot][half][lane] x 4 floats; then the heads' maxima
  constexpr int kRowWaves = kAlone ? 4 : 8;
  __shared__ float tab[kRowWaves][2][kMaxPairs];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const QKAxesArgs::Part p = a.part[blockIdx.y];
  if (p.heads == 0) return;
  const int D = 16 << a.unit_shift;
  const int64_t row0 = (int64_t)blockIdx.x * kRowWaves, row = row0 + wave;
  // the lane's place in its heads, its first head, heads from one of its runs (units) to the next
  const int shift = kHalves ? a.unit_shift : a.unit_shift + 1;
  const int u = lane & ((1 << shift) - 1), h0 = lane >> shift, step = 64 >> shift;
  const bool turn = kHalves ? u < a.rot_units : u < 2 * a.rot_units;
  constexpr int kRuns = 2 * NU;
  // channel in its head of run slot i, and its head
  const int c0 = kHalves ? (turn ? 8 * u : 16 * u) : 8 * u, c1 = kHalves ? (turn ? a.half + 8 * u : 16 * u + 8) : 8 * u;
  const auto chan = [&](int i) { return kHalves && (i & 1) ? c1 : c0; };
  const auto head = [&](int i) { return h0 + (kHalves ? i >> 1 : i) * step; };
  const auto has = [&](int i) { return kWhole || head(i) < p.heads; };
  const auto past = [&](int i) { return !kWhole && (kHalves ? i >> 1 : i) * step >= p.heads; };  // no lane has run i (few heads beside many)

  const int64_t from = min(row, a.T - 1);  // (the loads do not wait to know whether the row has a request)
  u32x4 x[kRuns];
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    x[i] = u32x4{0u, 0u, 0u, 0u};
    if (has(i)) x[i] = *reinterpret_cast<const u32x4*>(p.x + from * p.ts + head(i) * p.hs + chan(i));
  }
  // the workgroup's requests (one a lane); every wave comes to the same decision
  const int theirs = lane >= kRowWaves || row0 + lane >= a.T ? -1 : a.ids ? a.ids[row0 + lane] : 0;
  const uint64_t alive = __ballot((uint32_t)theirs < (uint32_t)a.requests);
  const int first = alive ? __builtin_amdgcn_readlane(theirs, __builtin_ctzll(alive)) : -1;
  const bool one = __ballot(theirs == first) == alive;
  const bool live = alive >> wave & 1;
  float own[kHalves ? 2 : 1][8];  // the weight of a norm per head: the same for all of the lane's heads
  const bool each = a.norm == WANMI_QKNORM_PER_HEAD;
  if (each) {
#pragma unroll
    for (int r = 0; r < (kHalves ? 2 : 1); ++r)
#pragma unroll
      for (int j = 0; j < 8; ++j) own[r][j] = p.gamma ? p.gamma[chan(r) + j] : 1.0f;
  }
  const bool across = !kAlone && a.norm == WANMI_QKNORM_ACROSS_HEADS && p.gamma;
  if (across) {
    const u32x4 rg = buffer_rsrc(p.gamma, 4u * (uint32_t)(p.heads * D));  // heads past the end: zeros, not used
    const uint32_t base = lds_addr(gam);
#pragma unroll
    for (int k = 0; k < 2 * kRuns; ++k)
      if (k % kRowWaves == wave)
        lds_dma_b128(rg, (uint32_t)((head(k >> 1) * D + chan(k >> 1) + 4 * (k & 1)) * 4), base + k * 1024);
  }
  float* maxima = gam + (a.norm == WANMI_QKNORM_ACROSS_HEADS ? 2 * kRuns * 256 : 0);
  const bool bound = !kAlone && a.kmax && blockIdx.y == 1;
  if (bound)
    for (int h = threadIdx.x; h < p.heads; h += 64 * kRowWaves) maxima[h] = 0.0f;
  float* tc = tab[wave][0];
  float* tsn = tab[wave][1];
  for (int i = lane; i < a.pairs; i += 64) {
    const int64_t at = from * a.axes + a.axis[i];
    const double pos = a.pos_float ? (double)reinterpret_cast<const float*>(a.pos)[at]
                                   : (double)reinterpret_cast<const int32_t*>(a.pos)[at];
    float sn, cs;
    sincos_turns(pos * a.turns[i], sn, cs);
    tc[i] = cs;
    tsn[i] = sn;
  }
  if (across || bound) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    __syncthreads();
  } else {  // nothing that other waves wrote
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  uint16_t* po = p.out + row * p.out_ts;
  if (live) {
    constexpr int kAngles = kHalves ? 8 : 4;
    float cs[kAngles], sn[kAngles];
#pragma unroll
    for (int j = 0; j < kAngles; ++j) {
      cs[j] = turn ? tc[kAngles * u + j] : 1.0f;
      sn[j] = turn ? tsn[kAngles * u + j] : 0.0f;
    }
    float rs = 1.0f;
    if (a.norm == WANMI_QKNORM_ACROSS_HEADS) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = bf16_lo(x[i][j]) * bf16_lo(x[i][j]) + bf16_hi(x[i][j]) * bf16_hi(x[i][j]);
        ss += (q[0] + q[1]) + (q[2] + q[3]);
      }
      rs = rsqrt_f32(wave_sum_f32_asc(ss) / (float)(p.heads * D) + a.eps);
      // (the row is unpacked anew below instead of being held as fp32)
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w = x[i][j];
          asm volatile("" : "+v"(w));
          x[i][j] = w;
        }
    }
#pragma unroll
    for (int i = 0; i < kRuns; i += kHalves ? 2 : 1) {
      if (past(i)) break;
      constexpr int kN = kHalves ? 2 : 1;  // runs taken together
      float v[kN][8];
#pragma unroll
      for (int r = 0; r < kN; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[r][2 * j] = bf16_lo(x[i + r][j]), v[r][2 * j + 1] = bf16_hi(x[i + r][j]);
      if (each) {
        float ss = 0.0f;
#pragma unroll
        for (int r = 0; r < kN; ++r) {
          float q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) q[j] = v[r][2 * j] * v[r][2 * j] + v[r][2 * j + 1] * v[r][2 * j + 1];
          ss += (q[0] + q[1]) + (q[2] + q[3]);
        }
        const float g = rsqrt_f32(head_sum(ss, shift) / (float)D + a.eps);
#pragma unroll
        for (int r = 0; r < kN; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[r][j] *= g * own[r][j];
      } else if (across) {
#pragma unroll
        for (int r = 0; r < kN; ++r) {
          const f32x4 lo = reinterpret_cast<const f32x4*>(gam)[(i + r) * 128 + lane], hi = reinterpret_cast<const f32x4*>(gam)[(i + r) * 128 + 64 + lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[r][j] *= rs * lo[j], v[r][4 + j] *= rs * hi[j];
        }
      } else if (a.norm == WANMI_QKNORM_ACROSS_HEADS) {
#pragma unroll
        for (int r = 0; r < kN; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[r][j] *= rs;
      }
      if (turn) {
        if constexpr (kHalves) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float s = v[0][j], t = v[1][j];
            v[0][j] = s * cs[j] - t * sn[j];
            v[1][j] = s * sn[j] + t * cs[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float s = v[0][2 * j], t = v[0][2 * j + 1];
            v[0][2 * j] = s * cs[j] - t * sn[j];
            v[0][2 * j + 1] = s * sn[j] + t * cs[j];
          }
        }
      }
      if (bound) {
        float ss = 0.0f;
#pragma unroll
        for (int r = 0; r < kN; ++r)
#pragma unroll
          for (int j = 0; j < 8; ++j) ss += v[r][j] * v[r][j];
        // a rounding to bf16 adds at most 2^-8 of a value: the written row's norm is below this
        const float n = sqrtf(head_sum(ss, shift)) * 1.00390625f;
        if (u == 0 && has(i)) {
          if (one) atomicMax(reinterpret_cast<unsigned int*>(maxima) + head(i), __float_as_uint(n));
          else raise_max(a.kmax + (int64_t)__builtin_amdgcn_readlane(theirs, wave) * p.heads + head(i), n);
        }
      }
#pragma unroll
      for (int r = 0; r < kN; ++r) {
        const u32x4 o = {pack_bf16x2(v[r][0], v[r][1]), pack_bf16x2(v[r][2], v[r][3]), pack_bf16x2(v[r][4], v[r][5]), pack_bf16x2(v[r][6], v[r][7])};
        if (has(i + r)) store_b128_guarded(o, po + head(i + r) * p.out_hs + chan(i + r));
      }
    }
  } else if (a.zero_rest && row < a.T) {
#pragma unroll
    for (int i = 0; i < kRuns; ++i)
      if (has(i)) store_b128_guarded(u32x4{0u, 0u, 0u, 0u}, po + head(i) * p.out_hs + chan(i));
  }
  if (bound && one && alive) {
    __syncthreads();
    for (int h = threadIdx.x; h < p.heads; h += 64 * kRowWaves) raise_max(a.kmax + (int64_t)first * p.heads + h, maxima[h]);
  }
}

__global__ __launch_bounds__(256) void qk_axes_zero_kernel(float* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0.0f;
}

// One instantiation for Q and K: the larger part's.
template <int NU, bool kHalves, bool kAlone>
void launch_qk_axes(const QKAxesArgs& a, hipStream_t s) {
  constexpr int kRowWaves = kAlone ? 4 : 8;
  const dim3 grid((unsigned)((a.T + kRowWaves - 1) / kRowWaves), a.part[1].heads ? 2u : 1u);
  const int per_head = 1 << a.unit_shift;
  const bool whole = a.part[0].heads * per_head == 64 * NU && (!a.part[1].heads || a.part[1].heads * per_head == 64 * NU);
  const int bytes = kAlone ? 0 : (a.norm == WANMI_QKNORM_ACROSS_HEADS ? 4096 * NU : 0) + (a.kmax ? 4 * a.part[1].heads : 0);
  // (16 units, more than 8192 channels: past the 64 KB that a launch has by itself, with the angles)
  if (NU == 16) {
    static int allowed[64] = {0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64 || !allowed[dev]) {
      for (const void* f : {reinterpret_cast<const void*>(&qk_axes_kernel<NU, kHalves, true, kAlone>), reinterpret_cast<const void*>(&qk_axes_kernel<NU, kHalves, false, kAlone>)})
        if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024) != hipSuccess) return;  // (the error is the launch's)
      if (dev >= 0 && dev < 64) allowed[dev] = 1;
    }
  }
  if (whole) hipLaunchKernelGGL((qk_axes_kernel<NU, kHalves, true, kAlone>), grid, dim3(64 * kRowWaves), bytes, s, a);
  else hipLaunchKernelGGL((qk_axes_kernel<NU, kHalves, false, kAlone>), grid, dim3(64 * kRowWaves), bytes, s, a);
}

template <bool kHalves>
void launch_qk_axes(const QKAxesArgs& a, int nu, hipStream_t s) {
  // Short rows that share nothing: many small workgroups (7799 rows of 32 + 4 heads of 64,
  // halves: 22.7 us; as eight rows a workgroup in the kernel that can share, with its registers, 25.9).
  const bool alone = !a.kmax && (a.norm != WANMI_QKNORM_ACROSS_HEADS || (!a.part[0].gamma && !a.part[1].gamma));
  if (nu <= 1 && alone) launch_qk_axes<1, kHalves, true>(a, s);
  else if (nu <= 2 && alone) launch_qk_axes<2, kHalves, true>(a, s);
  else if (nu <= 1) launch_qk_axes<1, kHalves, false>(a, s);
  else if (nu <= 2) launch_qk_axes<2, kHalves, false>(a, s);
  else if (nu <= 3) launch_qk_axes<3, kHalves, false>(a, s);
  else if (nu <= 4) launch_qk_axes<4, kHalves, false>(a, s);
  else if (nu <= 5) launch_qk_axes<5, kHalves, false>(a, s);
  else if (nu <= 6) launch_qk_axes<6, kHalves, false>(a, s);
  else if (nu <= 8) launch_qk_axes<8, kHalves, false>(a, s);
  else launch_qk_axes<16, kHalves, false>(a, s);
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
  // (a wave a row: a launch has fewer than 2^32 lanes)
  WANMI_REQUIRE(T >= 0 && T <= (1LL << 26) - 8, WANMI_ERR_ARG, "%s: T=%lld must be in [0, 2^26 - 8]", f, (long long)T);
  WANMI_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256, WANMI_ERR_UNSUPPORTED,
                "%s: head_dim=%d must be 32, 64, 128 or 256", f, head_dim);
  WANMI_REQUIRE(rope_pairs == WANMI_ROTATE_INTERLEAVED || rope_pairs == WANMI_ROTATE_HALVES, WANMI_ERR_ARG,
                "%s: unknown rope_pairs %d", f, rope_pairs);
  WANMI_REQUIRE(norm == WANMI_QKNORM_NONE || norm == WANMI_QKNORM_PER_HEAD || norm == WANMI_QKNORM_ACROSS_HEADS,
                WANMI_ERR_ARG, "%s: unknown norm %d", f, norm);
  WANMI_REQUIRE(eps >= 0.0f, WANMI_ERR_ARG, "%s: eps must be >= 0", f);
  WANMI_REQUIRE(axes >= 0 && axes <= 8 && (!axes || (axis_dims && freqs)), WANMI_ERR_ARG, "%s: at most 8 axes with their widths and frequencies", f);
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
  const int64_t bounds = k_maxnorm ? requests * k_heads : 0;
  WANMI_REQUIRE(bounds < (1LL << 31), WANMI_ERR_ARG, "%s: %lld requests of %d heads are too many", f, (long long)requests, k_heads);
  hipStream_t s = (hipStream_t)stream;
  const auto clear_bounds = [&]() {
    if (!bounds) return (int)WANMI_OK;
    hipLaunchKernelGGL(qk_axes_zero_kernel, dim3((unsigned)((bounds + 255) / 256)), dim3(256), 0, s, k_maxnorm, bounds);
    return check_launch(f);
  };
  if (T == 0) return clear_bounds();
  WANMI_REQUIRE(q && (positions || !rot) && q_out && (!k_heads || (k && k_out)), WANMI_ERR_ARG, "%s: null pointer", f);
  const int64_t strides[8] = {q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride,
                              k_heads ? k_token_stride : 0, k_heads ? k_head_stride : 0, k_heads ? k_out_token_stride : 0,
                              k_heads ? k_out_head_stride : 0};
  for (int64_t v : strides)
    WANMI_REQUIRE(v >= 0 && v % 8 == 0, WANMI_ERR_ARG, "%s: strides must be multiples of 8 elements, got %lld", f, (long long)v);
  for (const void* p : {q, (const void*)q_out, k, (const void*)k_out})
    WANMI_REQUIRE(((uintptr_t)p % 16) == 0, WANMI_ERR_ARG, "%s: tensors must be 16-byte aligned", f);
  // (read 16 bytes a lane, straight into LDS; a head's own weight is read by the element)
  for (const float* p : {q_gamma, k_gamma})
    WANMI_REQUIRE(norm != WANMI_QKNORM_ACROSS_HEADS || ((uintptr_t)p % 16) == 0, WANMI_ERR_ARG,
                  "%s: the weights of a norm across heads must be 16-byte aligned", f);
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
  const int cleared = clear_bounds();
  if (cleared != WANMI_OK) return cleared;
  const int units = (k_heads > q_heads ? k_heads : q_heads) * (head_dim / 16);
  const int nu = (units + 63) / 64;
  if (rope_pairs == WANMI_ROTATE_HALVES) launch_qk_axes<true>(a, nu, s);
  else launch_qk_axes<false>(a, nu, s);
  return check_launch(f);
}
