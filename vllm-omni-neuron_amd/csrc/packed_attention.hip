// Attention of packed rows over packed texts for gfx950, bf16 MFMA with fp32 softmax and sums.
//
//   o_i = sum_j exp(s q_i.k_j + b(j - i) - m_i) v_j / sum_j exp(s q_i.k_j + b(j - i) - m_i)
//
// The queries of request r are rows [q_off[r], q_off[r + 1]) of the batch, its keys and values rows [k_off[r],
// k_off[r + 1]) of the texts: all requests in one launch, nothing padded between them. b is absent (cross-attention) or a
// learned bias of the head for the bucket of the distance j - i (a text encoder's self-attention). A request without
// keys gives zeros. The offsets are read on the GPU and held inside the tensors, so that no offset reads or writes
// out of bounds; ascending ones that start at 0 are the caller's part.
//
// A workgroup of four waves takes one head of one tile of a request's rows: 128 rows, 32 per wave, all waves over the same
// keys (kSplit 1), or 32 rows with the keys shared out over the waves and their parts joined through LDS at the end
// (kSplit 4: few tiles of rows, over long texts). K and V pass through LDS in tiles of 64 (128) keys, loaded straight into it while the
// tile before is computed. S^T = K Q^T puts a row's scores into one lane (and lane ^ 32), so that the softmax is lane-local, and
// its P^T is the operand of O^T = V^T P^T as it stands. V stays [key][d] in LDS; its columns are read by the transposing LDS read
// (ds_read_b64_tr_b16: 16 lanes read four keys x 16 d and get one d's four keys each).
//
// The maximum m of a row is one that its running maximum may exceed by 2^8 before sums and outputs are rescaled: P then reaches
// 2^8 instead of 1, which costs bf16 and fp32 no precision, and nearly every tile after the first goes without a rescale.
//
// What bounds it: with many rows, a SIMD's matrix pipe and its VALU, which here run one after the other more than beside one another. 32760 rows of 40 heads x
// 128 over 512 and fewer keys (251 GFLOP, 687 MB) take 317 to 341 us (740 to 790 TFLOP/s): the matrix pipe is busy 39% of the cycles, the VALU 42%, LDS
// 24% (6% of that on bank conflicts). A score of 64 lanes costs the VALU 18 cycles (2^x 8.4, the multiply-add before it 2.7, conversion, sum and maximum 2.3
// each) beside 32 of MFMA at D = 128 and 16 at D = 64. 64 keys more cost 37 us there (1160 TFLOP/s), the rows themselves 92 (q and o, 671 MB); 1024 keys
// reach 1000 TFLOP/s, 8192 rows of 64 heads x 64 over 2048 keys 930; prompts of 6001 tokens with a bias there (159 GFLOP) take 195 to 213 us. With few rows it
// is the chain of launch, offsets, the tiles that one CU loads, and join: 16 rows of 40 heads over 512 keys 8.9 us for 11 MB.
// The constant-max kernel of attention.hip reaches 1340 TFLOP/s on long sequences with the same products and exponentials: eight waves of 32 rows over a ring of four
// tiles, loads of K and V apart, wave priorities by step. That scheme as a whole is not tried here. What did not help by itself (512 keys, 380 us): scores of a
// tile beside the softmax of the one before (443), workgroups that stay and load ahead for their next tile of rows (448), three workgroups a CU with tiles
// of 32 keys (386), half of the first workgroups held back or wave priorities (within 1%).
#include "packed_attention_plan.h"
#include "wanmi_common.h"

#include <algorithm>

namespace wanmi {

constexpr int kMaxSide = 128;         // bias buckets of one direction
constexpr int kMaxSaturation = 1024;  // the distance from which on a direction's last bucket holds
constexpr float kSlack = 8.0f;        // log2 units
constexpr float kBiasMax = 1e30f;     // of a finite bias, in units of the scores before their scale: beyond, scores vanish beside it
// A weight is 2^(s c - m c), by one multiply-add with the rounded m c. The rounding is up to 2^-24 of it: the same for all keys under one m, but not for
// tiles or waves with another, and where |m c| reaches 2^31 (scores in the thousands of millions; a row of nothing but a mask's lowest value) the rounding alone
// leaves the range of 2^x. Beyond this |m c|, where it is 2^-10 log2 units, m is subtracted from a row's scores instead, which is exact near the maximum.
constexpr float kFar = 16384.0f;

struct PackedAttnArgs {
  const uint16_t* q;  // row i, head h at q + i * q_ss + h * q_hs
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_ss, q_hs, k_ss, k_hs, v_ss, v_hs;
  const int* q_off;  // [requests + 1]
  const int* k_off;
  int requests;
  int T, Tk;
  int heads, group;   // query heads, and how many of them share a key head
  float scale_log2;   // s log2(e)
  float slack;        // kSlack / scale_log2
  float inv_scale;    // 1 / s
  void* out;          // bf16 [T, heads * D], or e4m3 codes
  int64_t o_ss;
  uint8_t* out_scales;  // MX: [T, heads * D / 32]
  int zero_rest;        // rows behind the last request: written as zeros, or left
  int tiles, per_xcd;   // tiles of rows (an upper bound), workgroups per XCD
  int together;         // heads that take the same tile one after the other; divides heads
};

// Distances of a head's bias in LDS: -(sat + 63) .. sat + 63.
__host__ __device__ constexpr int bias_entries(int sat) { return 2 * (sat + 63) + 1; }

struct BiasArgs {
  const void* table;  // [buckets, heads], fp32 or bf16
  int bf16;
  int side;           // buckets of one direction
  int both;           // buckets for later keys follow those for earlier ones; else every later key takes bucket 0
  int sat;            // the distance from which on the last bucket holds
  uint8_t bucket[kMaxSaturation + 1];  // of every distance up to there
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float max_lane_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// LDS tiles of K and V: rows of D bf16, 16-byte chunk c of a key's row in slot c ^ f(key). K is read 16 keys to a cycle,
// one chunk of each; V four keys to a cycle, 64 bytes of each: f spreads both over all banks.
template <int D>
__device__ __forceinline__ int k_slot(int key) {
  return D == 128 ? key & 15 : (key & 7) ^ ((key >> 3) & 1);
}
template <int D>
__device__ __forceinline__ int v_slot(int key) {
  return D == 128 ? (key & 3) << 2 : ((key >> 1) & 1) << 2;
}

// The tile `t` of the launch: its request, rows and keys. Every wave finds it for itself, 64 requests at a time. The rows behind the last
// request are one more request, without keys. False: no rows.
template <int kRows>
__device__ __forceinline__ bool find_tile(const PackedAttnArgs& a, int t, int& row0, int& rows, int& in_request, int& k0, int& keys) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int c = 0; c <= a.requests; c += 64) {
    const int r = min(c + lane, a.requests);
    const int next = min(r + 1, a.requests);
    const int q_lo = a.q_off[r], q_hi = a.q_off[next], k_lo = a.k_off[r], k_hi = a.k_off[next];  // (all four under way together)
    const int lo = min(max(q_lo, 0), a.T);
    int hi = r < a.requests ? min(max(q_hi, 0), a.T) : a.zero_rest ? a.T : lo;
    if (c + lane > a.requests) hi = lo;
    // inclusive sums over the lanes: within rows of 16, then each row's last into the rows behind it
    int sum = max(hi - lo + kRows - 1, 0) / kRows;
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xF, 0xF, false);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xF, 0xF, false);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xF, 0xF, false);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
    sum += before;
    const uint64_t hit = __ballot(sum > t);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int first = l ? __builtin_amdgcn_readlane(sum, l - 1) : before;
      const int at = __builtin_amdgcn_readlane(lo, l), end = __builtin_amdgcn_readlane(hi, l);
      in_request = (t - first) * kRows;
      if (in_request < 0 || in_request >= end - at) return false;
      row0 = at + in_request;
      rows = min(kRows, end - row0);
      // (the rows behind the last request: k_lo and k_hi are the same)
      const int kl = min(max(k_lo, 0), a.Tk), kn = max(min(max(k_hi, 0), a.Tk) - kl, 0);
      k0 = __builtin_amdgcn_readlane(kl, l);
      keys = __builtin_amdgcn_readlane(kn, l);
      return true;
    }
    before = __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// Rows of the output for a wave's stores: those past the extent are dropped. (Address and extent are the same in every lane, which the compiler
// does not prove: kept in vector registers each store would be a loop over the lanes' values.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(void* p, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at), hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), (short)0, (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// 16 outputs of a lane (d = 8 g + 4 hq + q of a block of 32) as bf16 pairs; kMx: as four words of codes and the block's
// scale byte. The block's other half is lane ^ 32's.
__device__ __forceinline__ int mx_codes(const uint32_t (&pp)[8], uint32_t (&codes)[4]) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 mag = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, pp[i] & 0x7FFF7FFFu));
  const int e = max_with_lane_xor32((int)(max(mag[0], mag[1]) >> 7));
  const int sx = max(e - 7, 0);
  const float sc = __uint_as_float((uint32_t)sx << 23);
#pragma unroll
  for (int g = 0; g < 4; ++g) codes[g] = cvt_e4m3x4_scaled(pp[2 * g], pp[2 * g + 1], sc);
  return sx;
}

// LDS of a workgroup without its bias: the ring of tiles; kSplit 4: the waves' rings, or the parts that are joined.
template <int D, int kSplit>
constexpr int ring_bytes() {
  constexpr int kRing = 2 * 2 * (kSplit == 4 ? 4 * 32 : 64) * 2 * D, kJoin = kSplit == 4 ? kSplit * 32 * (D * 4 + 8) : 0;
  return kRing > kJoin ? kRing : kJoin;
}

template <int D, bool kBias, int kSplit, bool kMx>
__global__ __launch_bounds__(256, 2) void packed_attention_kernel(PackedAttnArgs a, BiasArgs bias) {
  constexpr int kRows = 128 / kSplit;              // rows of a workgroup
  static_assert(kSplit == 1 || kSplit == 4, "whole waves of rows or of keys");
  constexpr bool kOwn = kSplit == 4;               // tiles of 32 keys, a wave's own; else 64 keys, of the workgroup
  constexpr int kHalves = kOwn ? 1 : 2;            // 32-key halves of a tile
  constexpr int kKeys = kOwn ? 32 : 64;
  constexpr int kRowB = 2 * D;                     // bytes
  constexpr int kChunks = D / 8;
  constexpr int kTile = kKeys * kRowB;             // of K, and as much of V
  constexpr int kLoads = kTile / (kOwn ? 1024 : 4096);  // per wave, of each
  constexpr int kRing = 2;
  static_assert(kRing * 2 * kTile * (kOwn ? 4 : 1) <= ring_bytes<D, kSplit>(), "the ring");
  // (not of a size that the compiler knows: with one workgroup a CU it would take accumulation registers for the products, and copy
  // scores and outputs from and to them; a head's bias behind it, for as many distances as its table tells apart)
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  [[maybe_unused]] float* sbias = reinterpret_cast<float*>(lds + ring_bytes<D, kSplit>());
  __shared__ __attribute__((aligned(1024))) uint8_t squery[kOwn ? 32 * kRowB : 16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hq = lane >> 5;
  // XCD x takes a contiguous run of (group of heads, tile, head): the tiles of a head read the same keys from its L2, and the heads of a
  // tile neighbouring parts of its rows. 32760 rows of 40 heads x 128, us with an eighth of the heads in a group against one: 64 keys 134 / 151,
  // 512 keys 380 / 389, 1024 keys 689 / 694; 64 heads x 64: alike.
  const int in_xcd = blockIdx.x >> 3;
  const int work = (int)(blockIdx.x & 7) * a.per_xcd + in_xcd;
  if (in_xcd >= a.per_xcd || work >= a.tiles * a.heads) return;
  const int group = work / (a.tiles * a.together), in_group = work - group * (a.tiles * a.together);
  const int tile = in_group / a.together, head = group * a.together + (in_group - tile * a.together);

  // ---- the head's bias over the distances -(sat + 63) .. sat + 63, over the scale: added to the scores before it. Its loads run beside
  // those of the offsets ----
  [[maybe_unused]] const int sat = bias.sat;
  if constexpr (kBias) {
    for (int i = threadIdx.x; i < bias_entries(sat); i += 256) {
      const int d = i - (sat + 63);
      int b = bias.bucket[min(abs(d), sat)];
      if (d > 0) b = bias.both ? b + bias.side : 0;
      const int at = b * a.heads + head;
      const float x = bias.bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(bias.table)[at]) : reinterpret_cast<const float*>(bias.table)[at];
      // (the lowest value of a type, as a mask has it, stays finite: a row of nothing else weighs all alike)
      sbias[i] = fabsf(x) < INFINITY ? fminf(fmaxf(x * a.inv_scale, -kBiasMax), kBiasMax) : x;
    }
  }
  int row0, rows, in_request, k0, keys;
  if (!find_tile<kRows>(a, tile, row0, rows, in_request, k0, keys)) return;

  const int lrow = lane / kChunks, lslot = lane % kChunks;
  constexpr int kPer = 64 / kChunks;  // rows of a load: four, or at D = 64 eight
  uint8_t* ring = lds + (kOwn ? wave * (kRing * 2 * kTile) : 0);
  const int qw = kOwn ? 0 : wave * 32;  // the wave's first row in the tile

  // ---- the wave's 32 queries, whole rows into LDS: into the second slot, which the second tile takes later; kSplit 4: all waves have the
  // same, eight rows are each one's part (gathered into the MFMA's layout from memory a load touches 32 bytes of 32 rows) ----
  uint8_t* sq = kOwn ? squery : lds + 2 * kTile + wave * (32 * kRowB);
  static_assert(kOwn || 4 * 32 * kRowB <= 2 * kTile, "the queries fit a slot");
  {
    const int live = min(rows - qw, 32);  // rows behind them read as zeros, and are not written
    const u32x4 r = buffer_rsrc(a.q + (int64_t)(row0 + qw) * a.q_ss + (int64_t)head * a.q_hs, live > 0 ? (uint32_t)(((live - 1) * a.q_ss + D) * 2) : 0u);
    constexpr int kN = 32 / kPer / (kOwn ? 4 : 1);
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const int first = ((kOwn ? wave * kN : 0) + j) * kPer, row = first + lrow;
      lds_dma_b128(r, (uint32_t)__umul24((uint32_t)row, (uint32_t)(a.q_ss * 2)) + (uint32_t)((lslot ^ k_slot<D>(row)) << 4), lds_addr(sq) + first * kRowB);
    }
  }

  // ---- loads of a tile of keys; kSplit 4: the wave's own keys into its own LDS ----
  const int khead = head / a.group;
  const uint16_t* kb = a.k + (int64_t)k0 * a.k_ss + (int64_t)khead * a.k_hs;
  const uint16_t* vb = a.v + (int64_t)k0 * a.v_ss + (int64_t)khead * a.v_hs;
  // the tile's number along the keys, and how many there are for this wave
  auto tile_at = [&](int t) { return kOwn ? t * kSplit + wave : t; };
  const int all = (keys + kKeys - 1) / kKeys;
  const int tiles = kOwn ? (all - wave + kSplit - 1) / kSplit : all;
  auto load_tile = [&](int t) {
    const int first = tile_at(t) * kKeys, left = min(keys - first, kKeys);  // > 0
    const u32x4 rk = buffer_rsrc(kb + (int64_t)first * a.k_ss, (uint32_t)(((left - 1) * a.k_ss + D) * 2));
    const u32x4 rv = buffer_rsrc(vb + (int64_t)first * a.v_ss, (uint32_t)(((left - 1) * a.v_ss + D) * 2));
    const uint32_t to = lds_addr(ring) + (uint32_t)((t % kRing) * 2 * kTile);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int r = ((kOwn ? 0 : wave * kLoads) + j) * kPer;  // the instruction's first row; keys past the text read as zeros
      const int key = r + lrow;
      lds_dma_b128(rk, (uint32_t)__umul24((uint32_t)key, (uint32_t)(a.k_ss * 2)) + (uint32_t)((lslot ^ k_slot<D>(key)) << 4), to + r * kRowB);
      lds_dma_b128(rv, (uint32_t)__umul24((uint32_t)key, (uint32_t)(a.v_ss * 2)) + (uint32_t)((lslot ^ v_slot<D>(key)) << 4), to + kTile + r * kRowB);
    }
  };
  if (tiles > 0) load_tile(0);
  if (kOwn && tiles > 1) load_tile(1);

  // ---- the queries as MFMA operands: lane holds d = 16 t + 8 hq .. + 7 of query col ----
  // (with the first tile, which is waited for here and not at the top of the loop)
  wait_vm<0>();
  if (kOwn || kBias) __syncthreads();
  bf16x8 qf[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) qf[t] = *reinterpret_cast<const bf16x8*>(sq + col * kRowB + (((2 * t + hq) ^ k_slot<D>(col)) << 4));
  wait_lgkm();  // (read before the second tile may come)

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
  float m = -INFINITY, sum = 0.0f;  // m in units of the scores before their scale
  float off = 0.0f;                 // -m c, rounded; 0 where there is no key above -inf yet (every P is 0), and where m is subtracted from the scores
  bool far = false, any_far = false;
  // (in a vector register: a multiply-add that reads a scalar one takes 4.5 cycles in place of 2.7)
  float c = a.scale_log2;
  asm volatile("" : "+v"(c));
  const bf16x2_t ones = {(__bf16)1.0f, (__bf16)1.0f};

  for (int t = 0; t < tiles; ++t) {
    if constexpr (!kOwn) {
      wait_vm<0>();
      __syncthreads();  // the tile is in LDS, and every wave is done with the one before it
      if (t + 1 < tiles) load_tile(t + 1);
    } else if (t + 1 < tiles) {
      wait_vm<2 * kLoads>();  // the next tile's may be under way
    } else {
      wait_vm<0>();
    }
    const uint8_t* tk = ring + (t % kRing) * 2 * kTile;
    const uint8_t* tv = tk + kTile;
    const int left = keys - tile_at(t) * kKeys;

    f32x16 s[kHalves];
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      const int key = 32 * i + col;
      const uint8_t* row = tk + key * kRowB;
      // register r of half i: key 32 i + 8 (r >> 2) + 4 hq + (r & 3). The products are added to the bias; where all of the half's distances
      // are beyond the last bucket's first they are all alike, and read from the table's end
      if constexpr (kBias) {
        const int d0 = tile_at(t) * kKeys + 32 * i - (in_request + qw);  // first key - first query
        const float* pb = sbias + (sat + 63 + min(max(d0, -(sat + 32)), sat + 32) + 4 * hq - col);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = pb[8 * (r >> 2) + (r & 3)];
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = 0.0f;
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const bf16x8 kf = *reinterpret_cast<const bf16x8*>(row + (((2 * d + hq) ^ k_slot<D>(key)) << 4));
        s[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[d], s[i], 0, 0, 0);
      }
    }
    if (left < 32 * kHalves) {
      asm volatile("");
      const int mine = left - 4 * hq;
#pragma unroll
      for (int i = 0; i < kHalves; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * i + 8 * (r >> 2) + (r & 3) >= mine) s[i][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      float h = s[i][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) h = fmaxf(h, s[i][r]);
      mx = fmaxf(mx, h);
    }
    mx = max_lane_xor32(mx);
    if (__any(mx > m + a.slack)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      off = m == -INFINITY ? 0.0f : -m * c;  // no key above -inf yet: every P is 0
      far = fabsf(off) > kFar;
      any_far = __any(far);
      if (far) off = 0.0f;
      if (t > 0) {  // (before, there is nothing to rescale)
        sum *= f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= f;
      }
    }
    if (any_far) {
      asm volatile("");
      const float from = far ? m : 0.0f;
#pragma unroll
      for (int i = 0; i < kHalves; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] -= from;
    }
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      bf16x8 pf[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i][8 * u + 2 * j], c, off));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[i][8 * u + 2 * j + 1], c, off));
          w[j] = pack_bf16x2(p0, p1);
          // The rounded weights, those that multiply V: their rounding, up to 2^-8 each and the same for keys of one score, then leaves a mean of equal values as
          // it is. One instruction a pair (by shifts and additions: 1024 keys 703 us in place of 687, prompts of 6001 tokens 203 in place of 194).
          sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w[j]), ones, sum, false);
        }
        pf[u] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // lane's keys: 16 u + 4 hq .. + 3 and 8 further, of d = 32 dt + col; it reads four d of key + (lane & 15) / 4
        const int key = 32 * i + 16 * u + 4 * hq + ((lane & 15) >> 2);
        const int ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        const uint8_t* p0 = tv + key * kRowB + 8 * (lane & 1);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
          const int at = ((4 * dt + ch) ^ v_slot<D>(key)) << 4;  // v_slot(key + 8) is the same
          typedef __attribute__((address_space(3))) s16x4* lds4;
          const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p0 + at));
          const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p0 + 8 * kRowB + at));
          const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[u], acc[dt], 0, 0, 0);
        }
      }
    }
    if (kOwn && t + 2 < tiles) {
      wait_lgkm();  // the wave has read its tile
      load_tile(t + 2);
    }
  }
  sum = add_lane_xor32(sum);

  if constexpr (!kOwn) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no keys: zeros; NaN stays
    // The slot that the last tile is not in: every wave is past the barrier behind its last use, and no load is under way to it.
    uint8_t* stage = lds + (tiles % kRing) * 2 * kTile + wave * (32 * kRowB);
    const int live = min(rows - qw, 32);  // rows of the wave
    [[maybe_unused]] uint32_t sbytes = 0;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      uint32_t pp[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) pp[i] = pack_bf16x2(acc[dt][2 * i] * inv, acc[dt][2 * i + 1] * inv);
      if constexpr (kMx) {
        uint32_t codes[4];
        sbytes |= (uint32_t)mx_codes(pp, codes) << (8 * dt);
#pragma unroll
        for (int g = 0; g < 4; ++g) {  // codes 32 dt + 8 g + 4 hq .. + 3
          const int chunk = 2 * dt + (g >> 1);
          *reinterpret_cast<uint32_t*>(stage + col * D + ((chunk ^ ((col >> 1) & (D / 16 - 1))) << 4) + 8 * (g & 1) + 4 * hq) = codes[g];
        }
      } else {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint2*>(stage + col * kRowB + (((4 * dt + g) ^ (col & (kChunks - 1))) << 4) + 8 * hq) = make_uint2(pp[2 * g], pp[2 * g + 1]);
      }
    }
    // (a wave's LDS operations complete in order: no barrier before its own rows are read back; rows behind the wave's are dropped)
    const int64_t item = kMx ? 1 : 2;
    const auto ro = row_rsrc(reinterpret_cast<uint8_t*>(a.out) + ((int64_t)(row0 + qw) * a.o_ss + head * D) * item, (uint32_t)max(live, 0) * (uint32_t)(a.o_ss * item));
    if constexpr (kMx) {
      constexpr int kPerRow = D / 16, kStep = 64 / kPerRow;
#pragma unroll
      for (int it = 0; it < 32 / kStep; ++it) {
        const int r = it * kStep + lane / kPerRow, chunk = lane % kPerRow;
        const u32x4 x = *reinterpret_cast<const u32x4*>(stage + r * D + ((chunk ^ ((r >> 1) & (D / 16 - 1))) << 4));
        __builtin_amdgcn_raw_buffer_store_b128(x, ro, (int)(__umul24((uint32_t)r, (uint32_t)a.o_ss) + chunk * 16), 0, 2);
      }
      if (hq == 0 && col < live) {
        uint8_t* ps = a.out_scales + (int64_t)(row0 + qw + col) * (a.heads * (D / 32)) + head * (D / 32);
        if constexpr (D == 128) *reinterpret_cast<uint32_t*>(ps) = sbytes;
        else *reinterpret_cast<uint16_t*>(ps) = (uint16_t)sbytes;
      }
    } else {
#pragma unroll
      for (int it = 0; it < 32 / kPer; ++it) {
        const int r = it * kPer + lrow;
        const u32x4 x = *reinterpret_cast<const u32x4*>(stage + r * kRowB + ((lslot ^ (r & (kChunks - 1))) << 4));
        __builtin_amdgcn_raw_buffer_store_b128(x, ro, (int)(__umul24((uint32_t)r, (uint32_t)(a.o_ss * 2)) + lslot * 16), 0, 2);
      }
    }
  } else {
    // ---- join the waves' parts: [wave][d][row] sums of P V, then [wave][row] maxima and sums ----
    __syncthreads();  // every wave is done with its tiles
    float* parts = reinterpret_cast<float*>(lds);
    float* stats = parts + kSplit * 32 * D;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) parts[(wave * D + 32 * dt + 8 * (r >> 2) + 4 * hq + (r & 3)) * 32 + col] = acc[dt][r];
    if (hq == 0) {
      stats[wave * 64 + col] = m;
      stats[wave * 64 + 32 + col] = sum;
    }
    __syncthreads();
    if (wave >= D / 32) return;
    float mw[kSplit], mm = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kSplit; ++w) mm = fmaxf(mm, mw[w] = stats[w * 64 + col]);
#pragma unroll
    for (int w = 0; w < kSplit; ++w) {
      mw[w] = mw[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw[w] - mm) * c);
      const float part = stats[w * 64 + 32 + col];
      total += part == 0.0f ? 0.0f : mw[w] * part;
    }
    // a NaN maximum is no maximum, but its sum is NaN
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    float o[16];  // d = 32 wave + 8 g + 4 hq + q of row col
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * wave + 8 * (r >> 2) + 4 * hq + (r & 3);
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kSplit; ++w) x = fmaf(mw[w], parts[(w * D + d) * 32 + col], x);
      o[r] = x * inv;
    }
    uint32_t pp[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) pp[i] = pack_bf16x2(o[2 * i], o[2 * i + 1]);
    const int64_t row = row0 + col;
    if constexpr (kMx) {
      uint32_t codes[4];
      const int sx = mx_codes(pp, codes);
      if (col < rows) {
        uint8_t* po = reinterpret_cast<uint8_t*>(a.out) + row * a.o_ss + head * D + 32 * wave + 4 * hq;
#pragma unroll
        for (int g = 0; g < 4; ++g) *reinterpret_cast<uint32_t*>(po + 8 * g) = codes[g];
        if (hq == 0) a.out_scales[row * (a.heads * (D / 32)) + head * (D / 32) + wave] = (uint8_t)sx;
      }
    } else if (col < rows) {
      uint16_t* po = reinterpret_cast<uint16_t*>(a.out) + row * a.o_ss + head * D + 32 * wave + 4 * hq;
#pragma unroll
      for (int g = 0; g < 4; ++g) *reinterpret_cast<uint2*>(po + 8 * g) = make_uint2(pp[2 * g], pp[2 * g + 1]);
    }
  }
}

template <int D, bool kBias, int kSplit>
static int launch(PackedAttnArgs a, const BiasArgs& b, hipStream_t stream, const char* what) {
  constexpr int kRows = 128 / kSplit;
  // every request ends in at most one part of a tile, and so do the rows behind the last
  const int64_t tiles = a.T / kRows + a.requests + 1;
  const int64_t per = (tiles * a.heads + 7) / 8;
  // (a launch has fewer than 2^32 lanes)
  WANMI_REQUIRE(tiles * a.heads < (1LL << 24) - 8, WANMI_ERR_ARG, "%s: %lld tiles of rows times %d heads are too many", what, (long long)tiles, a.heads);
  a.tiles = (int)tiles;
  a.per_xcd = (int)per;
  a.together = a.heads % 8 == 0 ? a.heads / 8 : 1;
  const unsigned lds = ring_bytes<D, kSplit>() + (kBias ? (unsigned)(bias_entries(b.sat) * sizeof(float)) : 0u);
  if constexpr (!kBias) {
    if (a.out_scales) {
      hipLaunchKernelGGL((packed_attention_kernel<D, kBias, kSplit, true>), dim3((unsigned)(8 * per)), dim3(256), lds, stream, a, b);
      return check_launch(what);
    }
  }
  hipLaunchKernelGGL((packed_attention_kernel<D, kBias, kSplit, false>), dim3((unsigned)(8 * per)), dim3(256), lds, stream, a, b);
  return check_launch(what);
}

template <bool kBias, int D>
static int dispatch(const PackedAttnArgs& a, const BiasArgs& b, hipStream_t stream, const char* what) {
  if (packed_keys_shared(a.T, a.Tk, a.requests, a.heads, D)) return launch<D, kBias, 4>(a, b, stream, what);
  return launch<D, kBias, 1>(a, b, stream, what);
}

// What both entry points check: sizes, strides and alignment that the kernel's 16-byte accesses and 32-bit offsets need.
static int check_args(const PackedAttnArgs& a, int64_t T, int64_t Tk, int64_t requests, int64_t heads, int64_t k_heads, int head_dim, const char* what) {
  WANMI_REQUIRE(head_dim == 64 || head_dim == 128, WANMI_ERR_UNSUPPORTED, "%s: head_dim %d is not 64 or 128", what, head_dim);
  WANMI_REQUIRE(T >= 0 && T < (1LL << 28) && Tk >= 0 && Tk < (1LL << 28), WANMI_ERR_ARG, "%s: %lld rows, %lld keys: at most 2^28 - 1", what, (long long)T, (long long)Tk);
  WANMI_REQUIRE(requests >= 0 && requests < (1 << 20), WANMI_ERR_ARG, "%s: %lld requests: at most 2^20 - 1", what, (long long)requests);
  WANMI_REQUIRE(heads > 0 && k_heads > 0 && heads % k_heads == 0 && heads <= 1024, WANMI_ERR_ARG, "%s: %lld heads (at most 1024) over %lld key heads", what, (long long)heads, (long long)k_heads);
  WANMI_REQUIRE(a.inv_scale >= 0x1p-24f && a.inv_scale <= 0x1p64f, WANMI_ERR_ARG, "%s: the scale must be in 2^-64 .. 2^24", what);
  // (rows enter the 24-bit products and 32-bit offsets of a tile; heads only 64-bit addresses)
  const int64_t rows[3] = {a.q_ss, a.k_ss, a.v_ss}, head[3] = {a.q_hs, a.k_hs, a.v_hs};
  for (int i = 0; i < 3; ++i) {
    WANMI_REQUIRE(rows[i] >= 0 && rows[i] % 8 == 0 && rows[i] < (1 << 22), WANMI_ERR_ARG, "%s: row stride %lld must be a multiple of 8 below 2^22", what, (long long)rows[i]);
    WANMI_REQUIRE(head[i] >= 0 && head[i] % 8 == 0 && head[i] < (1LL << 40), WANMI_ERR_ARG, "%s: head stride %lld must be a multiple of 8 below 2^40", what, (long long)head[i]);
  }
  if (T == 0) return WANMI_OK;
  WANMI_REQUIRE(a.q && a.out && a.q_off && a.k_off && (Tk == 0 || (a.k && a.v)), WANMI_ERR_ARG, "%s: null pointer", what);
  WANMI_REQUIRE(((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) % 16 == 0, WANMI_ERR_ARG, "%s: q, k, v and out must be 16-byte aligned", what);
  WANMI_REQUIRE(T == 1 || a.q_ss >= head_dim, WANMI_ERR_ARG, "%s: rows of q overlap", what);
  WANMI_REQUIRE(Tk <= 1 || (a.k_ss >= head_dim && a.v_ss >= head_dim), WANMI_ERR_ARG, "%s: rows of k or v overlap", what);
  WANMI_REQUIRE(a.o_ss % 16 == 0 && a.o_ss >= heads * head_dim && a.o_ss < (1 << 22), WANMI_ERR_ARG, "%s: the output's row stride must be a multiple of 16 of at least %lld, below 2^22", what, (long long)(heads * head_dim));
  return WANMI_OK;
}

}  // namespace wanmi

extern "C" int wanmi_packed_cross_attention(const void* q, int64_t q_ss, int64_t q_hs, const void* k, int64_t k_ss, int64_t k_hs,
                                            const void* v, int64_t v_ss, int64_t v_hs, const int* q_offsets, const int* k_offsets,
                                            int64_t requests, int64_t T, int64_t Tk, int64_t heads, int64_t k_heads, int head_dim,
                                            float scale, void* out, int64_t o_ss, uint8_t* out_scales, int zero_rest, void* stream) {
  using namespace wanmi;
  clear_error();
  PackedAttnArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, q_ss, q_hs, k_ss, k_hs, v_ss, v_hs, q_offsets, k_offsets, (int)requests,
                   (int)T, (int)Tk, (int)heads, (int)(k_heads > 0 ? heads / k_heads : 1), scale * 1.4426950408889634f, kSlack / (scale * 1.4426950408889634f), 1.0f / scale, out, o_ss, out_scales, zero_rest, 0, 0, 1};
  const int st = check_args(a, T, Tk, requests, heads, k_heads, head_dim, "wanmi_packed_cross_attention");
  if (st != WANMI_OK || T == 0) return st;
  const char* what = "wanmi_packed_cross_attention";
  return head_dim == 64 ? dispatch<false, 64>(a, BiasArgs{}, (hipStream_t)stream, what) : dispatch<false, 128>(a, BiasArgs{}, (hipStream_t)stream, what);
}

extern "C" int wanmi_relative_bias_attention(const void* q, int64_t q_ss, int64_t q_hs, const void* k, int64_t k_ss, int64_t k_hs,
                                             const void* v, int64_t v_ss, int64_t v_hs, const int* offsets, int64_t requests, int64_t T,
                                             int64_t heads, int head_dim, float scale, const void* table, int table_bf16,
                                             const int* starts, int side, int both, void* out, int64_t o_ss, int zero_rest, void* stream) {
  using namespace wanmi;
  clear_error();
  const char* what = "wanmi_relative_bias_attention";
  PackedAttnArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, q_ss, q_hs, k_ss, k_hs, v_ss, v_hs, offsets, offsets, (int)requests,
                   (int)T, (int)T, (int)heads, 1, scale * 1.4426950408889634f, kSlack / (scale * 1.4426950408889634f), 1.0f / scale, out, o_ss, nullptr, zero_rest, 0, 0, 1};
  const int st = check_args(a, T, T, requests, heads, heads, head_dim, what);
  if (st != WANMI_OK) return st;
  WANMI_REQUIRE(side >= 1 && side <= kMaxSide && starts, WANMI_ERR_ARG, "%s: %d buckets of one direction, at most %d", what, side, kMaxSide);
  for (int i = 0; i < side; ++i)
    WANMI_REQUIRE(starts[i] >= (i ? starts[i - 1] : 0) && starts[i] <= kMaxSaturation && starts[0] == 0, WANMI_ERR_ARG,
                  "%s: the buckets' first distances must ascend from 0 to at most %d", what, kMaxSaturation);
  BiasArgs b{table, table_bf16, side, both, starts[side - 1], {0}};
  for (int n = 0, i = 0; n <= b.sat; ++n) {
    while (i + 1 < side && starts[i + 1] <= n) ++i;
    b.bucket[n] = (uint8_t)i;
  }
  if (T == 0) return WANMI_OK;
  WANMI_REQUIRE(table, WANMI_ERR_ARG, "%s: null pointer", what);
  return head_dim == 64 ? dispatch<true, 64>(a, b, (hipStream_t)stream, what) : dispatch<true, 128>(a, b, (hipStream_t)stream, what);
}
