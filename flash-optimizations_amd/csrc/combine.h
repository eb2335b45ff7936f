// Merge of split partials with the sink, shared by the decodes: partial O / l and
// log2 l + m per (token, split, head), [tokens, splits, heads, 512] and [tokens,
// splits, heads] floats, to out (BF16) and lse. kNatural: the partials' coordinates
// in their own order and any number of heads (4-bit records, trees); otherwise in
// partial_coord() order with heads a multiple of 16 (Packed and Native). kRagged: of the
// slots of request r's tokens only the first counts[r] hold partials; none: its rows are
// finished already.
#pragma once
#include "remnant_device.h"

namespace {

using namespace rm;

constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Order of a split partial's 512 floats: coordinate 64 u + 16 q + c (u < 8, q <
// 4, c < 16) is at 64 u + 4 c + q, so the 16-coordinate stride at which a
// consumer lane holds its coordinates becomes four runs of four.
__device__ __forceinline__ constexpr int partial_coord(int at) {
  return (at & ~63) + 16 * (at & 3) + ((at & 63) >> 2);
}

// Butterfly over the wave's 64 lanes with the pairing of xor distances 1, 2,
// 4, ..., 32 (quad permutes, the half-row and row mirrors -- in a butterfly
// every lane of an aligned group already holds the same value, so the mirror
// partner gives the xor partner's value -- then the 16- and 32-lane swaps):
// the same additions as a shuffle-xor butterfly, without LDS round trips.
template <int kCtrl>
__device__ __forceinline__ float dpp_f(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xf, 0xf, false));
}
template <bool kMax>
__device__ __forceinline__ float wave_all(float x) {
  auto op = [](float u, float v) { return kMax ? fmaxf(u, v) : u + v; };
  x = op(x, dpp_f<0xB1>(x));   // quad_perm [1,0,3,2]
  x = op(x, dpp_f<0x4E>(x));   // quad_perm [2,3,0,1]
  x = op(x, dpp_f<0x141>(x));  // row_half_mirror
  x = op(x, dpp_f<0x140>(x));  // row_mirror
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  x = op(u2f(h[0]), u2f(h[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return op(u2f(q[0]), u2f(q[1]));
}
__device__ __forceinline__ float lane_of(float x, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
}

// Merge split partials with the sink, for many rows: one wave per (token,
// head) row, lane l owning the coordinates stored at 8l..8l+7. The partial loads
// of up to kWaveBatch splits are issued together with the split LSEs (lane s
// holds split s), so a row costs one round trip per kWaveBatch splits.
// kWaveBatch is 4 for up to four splits and 8 beyond. Loads past the last split
// repeat it and are left out of the sum (not added with weight zero: an infinite
// partial would become a NaN): a branch around each load would make the kernel,
// which runs once per row, mostly instruction fetch (traced, with the token and
// head from the grid instead of a division: 64 heads x 16 tokens 4.5 -> 4.1 us, 128
// heads 5.6 -> 4.9, 16 heads x 64 tokens of four splits 4.6 unchanged; the
// other combine, one token of 64 splits, 3.9 -> 3.4).
template <int kWaveBatch, bool kNatural, bool kRagged>
__global__ __launch_bounds__(256) void combine_wave_kernel(const float* __restrict__ ws_o,
                                                           const float* __restrict__ ws_lse,
                                                           const float* __restrict__ sink,
                                                           int slots, int heads,
                                                           uint16_t* __restrict__ out,
                                                           float* __restrict__ lse,
                                                           const int32_t* __restrict__ counts) {
  const int lane = wave_lane();
  // block (x, y, z): heads 4x .. 4x + 3 of token y (of request z, where they are ragged)
  const int64_t t = kRagged ? blockIdx.z * gridDim.y + blockIdx.y : blockIdx.y;
  const int h = blockIdx.x * 4 + uniform((int)(threadIdx.x >> 6));
  if (kNatural && h >= heads) return;
  const int splits = kRagged ? counts[blockIdx.z] : slots;
  if (kRagged && splits == 0) return;
  const int64_t row = t * heads + h;
  const float* src = ws_o + (t * slots * heads + h) * kHeadDim + 8 * lane;
  const int64_t step = (int64_t)heads * kHeadDim;
  f32x4 x[2 * kWaveBatch];
#pragma unroll
  for (int u = 0; u < kWaveBatch; ++u) {
    const float* const from = src + min(u, splits - 1) * step;
    x[2 * u] = *(const f32x4*)from;
    x[2 * u + 1] = *(const f32x4*)(from + 4);
  }
  const float lse_at = ws_lse[(t * slots + min(lane, splits - 1)) * heads + h];
  const float ls = lane < splits ? lse_at : -INFINITY;
  const float sink2 = sink ? sink[h] * kLog2e : -INFINITY;
  const float mz = wave_all<true>(fmaxf(ls, sink2));
  const float w = (mz != -INFINITY && lane < splits) ? exp2f(ls - mz) : 0.0f;
  const float z = wave_all<false>(w);
  f32x4 a0 = {0.f, 0.f, 0.f, 0.f}, a1 = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += kWaveBatch) {
    if (s0 > 0) {
#pragma unroll
      for (int u = 0; u < kWaveBatch; ++u) {
        const float* const from = src + min(s0 + u, splits - 1) * step;
        x[2 * u] = *(const f32x4*)from;
        x[2 * u + 1] = *(const f32x4*)(from + 4);
      }
    }
#pragma unroll
    for (int u = 0; u < kWaveBatch; ++u) {
      const int sp = s0 + u;
      if (sp >= splits) break;
      const float ww = lane_of(w, sp);
      a0 += ww * x[2 * u];
      a1 += ww * x[2 * u + 1];
    }
  }
  float lse_out = -INFINITY;
  f32x4 r0 = {0.f, 0.f, 0.f, 0.f}, r1 = {0.f, 0.f, 0.f, 0.f};
  if (mz != -INFINITY) {
    const float zt = z + exp2f(sink2 - mz);
    const float inv = 1.0f / zt;
    r0 = a0 * inv;
    r1 = a1 * inv;
    lse_out = (mz + log2f(zt)) * kLn2;
  }
  if constexpr (kNatural) {
    u32x4 o;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      o[q] = __builtin_bit_cast(uint32_t, bf16_pair(r0[2 * q], r0[2 * q + 1]));
      o[2 + q] = __builtin_bit_cast(uint32_t, bf16_pair(r1[2 * q], r1[2 * q + 1]));
    }
    *(u32x4*)(out + row * kHeadDim + 8 * lane) = o;
  } else {
    // r0[q] and r1[q] are neighbouring coordinates: partial_coord(8 lane + q) and + 1
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(uint32_t*)(out + row * kHeadDim + partial_coord(8 * lane + q)) =
          bf16_rne(r0[q]) | (bf16_rne(r1[q]) << 16);
  }
  if (lane == 0) lse[row] = lse_out;
}

// Merge split partials with the sink, for few rows (small batches). One
// workgroup (4 waves) per (token, head, 64-coordinate slice): lane l owns the
// coordinate stored at 64 slice + l; wave w takes
// splits w, w + 4, ... (<= 16 each, all loads in flight at once); the four
// partial sums meet in LDS in a fixed order. The split weights come from every
// split's LSE, read by every wave (lane s holds split s; splits <= 64).
// kPerWave (4, 8 or 16) is the smallest that covers the splits; loads past the
// last split repeat it and are left out of the sum, as in combine_wave_kernel.
constexpr int kCombineSlices = kHeadDim / 64;
template <int kPerWave, bool kNatural, bool kRagged>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ ws_o,
                                                      const float* __restrict__ ws_lse,
                                                      const float* __restrict__ sink, int slots,
                                                      int heads, uint16_t* __restrict__ out,
                                                      float* __restrict__ lse,
                                                      const int32_t* __restrict__ counts) {
  __shared__ float part[4][64];
  const int lane = wave_lane();
  const int wave = uniform((int)(threadIdx.x >> 6));
  // block (x, y, z): head x / 8 and slice x % 8 of token y (of request z)
  const int64_t t = kRagged ? blockIdx.z * gridDim.y + blockIdx.y : blockIdx.y;
  const int h = blockIdx.x / kCombineSlices;
  const int slice = blockIdx.x % kCombineSlices;
  const int splits = kRagged ? counts[blockIdx.z] : slots;
  if (kRagged && splits == 0) return;
  const int64_t row = t * heads + h;
  const int64_t step = (int64_t)heads * kHeadDim;
  const float* src = ws_o + (t * slots * heads + h) * kHeadDim + 64 * slice + lane;
  // issue every load first: this wave's partials and all split LSEs
  float x[kPerWave];
#pragma unroll
  for (int u = 0; u < kPerWave; ++u) {
    const int s = wave + 4 * u;
    x[u] = src[min(s, splits - 1) * step];
  }
  const float lse_at = ws_lse[(t * slots + min(lane, splits - 1)) * heads + h];
  const float ls = lane < splits ? lse_at : -INFINITY;
  const float sink2 = sink ? sink[h] * kLog2e : -INFINITY;
  const float mz = wave_all<true>(fmaxf(ls, sink2));
  const float w = (mz != -INFINITY && lane < splits) ? exp2f(ls - mz) : 0.0f;
  const float z = wave_all<false>(w);
  float acc = 0.0f;
#pragma unroll
  for (int u = 0; u < kPerWave; ++u) {
    const int s = wave + 4 * u;
    if (s < splits) acc += lane_of(w, s) * x[u];
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    float lse_out = -INFINITY, r = 0.0f;
    if (mz != -INFINITY) {
      const float zt = z + exp2f(sink2 - mz);
      const float inv = 1.0f / zt;
      r = (part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane]) * inv;
      lse_out = (mz + log2f(zt)) * kLn2;
    }
    const int at = 64 * slice + lane;
    if constexpr (kNatural)
      out[row * kHeadDim + at] = __builtin_bit_cast(uint16_t, (__bf16)r);
    else
      out[row * kHeadDim + partial_coord(at)] = (uint16_t)bf16_rne(r);
    if (lane == 0 && slice == 0) lse[row] = lse_out;
  }
}

template <bool kNatural, bool kRagged = false>
void launch_combine(const float* ws_o, const float* ws_lse, const float* sink, int slots,
                    int64_t tokens, int64_t heads, uint16_t* out, float* lse, hipStream_t s,
                    const int32_t* counts = nullptr, int64_t requests = 1) {
  // rows: one workgroup per 64 coordinates of each. In natural order also where the wave
  // form would take two turns (decode of 4-bit records, 16 tokens x 16 heads, 16 splits
  // 15.3 -> 13.1 us with it; 24 tokens, 8 splits: 16.8 with this form, 16.3 the other), but
  // not where most rows have fewer partials than slots
  const bool few = tokens * heads < 256 || (kNatural && !kRagged && slots > 8);
  const auto wave = slots <= 4 || kRagged ? combine_wave_kernel<4, kNatural, kRagged>
                                          : combine_wave_kernel<kRagged ? 4 : 8, kNatural, kRagged>;
  const auto kern = !few          ? wave
                    : slots <= 16 ? combine_kernel<4, kNatural, kRagged>
                    : slots <= 32 ? combine_kernel<8, kNatural, kRagged>
                                  : combine_kernel<16, kNatural, kRagged>;
  const dim3 grid((unsigned)(few ? heads * kCombineSlices : (heads + 3) / 4),
                  (unsigned)(tokens / requests), (unsigned)requests);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, ws_o, ws_lse, sink, slots, (int)heads, out, lse,
                     counts);
}

}  // namespace
