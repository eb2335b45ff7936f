// Store and reader of index records (index_device.h).
//
// Store: r = RN(1 / RN(sqrt(sum x^2 / 128 + eps))), n = bf16((x r) w), the last 64
// coordinates of n rotated by a frequency row and rounded to BF16 again, then codes
// n / 2^e under the smallest e with max(amax, 1e-4) <= 448 * 2^e. The sum takes 8
// neighbours in turn, then pairs of neighbours, so that every rounding is fixed.
// Reader: code * scale, rounded once to BF16.
//
// Both give a row to 16 lanes of 8 coordinates, four rows a wave and turn: reductions
// stay within a DPP row, and each access is the widest that a row allows.
// Bound by memory: 2^20 BF16 rows to random slots 105 us, read back 85.
#include <algorithm>

#include "index_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kWaves = 4;
// Rows of a launch of the store. A launch has fewer than 2^32 threads (2^28 rows): with more
// the count wraps, without an error.
constexpr int64_t kLaunchRows = (int64_t)1 << 27;

template <int kCtrl>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xf, 0xf, false));
}
template <int kCtrl>
__device__ __forceinline__ int dpp(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kCtrl, 0xf, 0xf, false);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E;  // quad permutes
constexpr int kHalfMirror = 0x141, kMirror = 0x140;

struct StoreArgs {
  const void* x;
  int64_t stride;
  const float* weight;
  float eps;
  const int32_t *slots, *position;
  const float* freqs;
  int64_t freq_rows, n;
  uint8_t* pool;
  int64_t pool_rows;
  uint32_t ratio;
};

template <bool kBf16>
__global__ __launch_bounds__(64 * kWaves) void index_store_kernel(StoreArgs a) {
  const int lane = wave_lane(), j = lane & 15;
  const int64_t i = ((int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6)) * 4 + (lane >> 4);
  if (i >= a.n) return;  // (rows are 16 lanes: no reduction crosses them)
  // The input does not wait for the slot, and is read where that turns out to be refused too
  // (2^20 rows of BF16, stored and read back: 186 us; 189 when it waited).
  const int32_t slot = a.slots[i], pos = a.freqs ? a.position[i] : 0;
  float v[8];
  if constexpr (kBf16) {
    const u32x4 raw = *(const u32x4*)((const uint16_t*)a.x + i * a.stride + 8 * j);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[2 * c] = u2f(raw[c] << 16);
      v[2 * c + 1] = u2f(raw[c] & 0xffff0000u);
    }
  } else {
    const f32x4* const at = (const f32x4*)((const float*)a.x + i * a.stride + 8 * j);
    const f32x4 lo = at[0], hi = at[1];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = lo[c], v[4 + c] = hi[c];
  }
  const f32x4 w0 = *(const f32x4*)(a.weight + 8 * j), w1 = *(const f32x4*)(a.weight + 8 * j + 4);
  const bool refused = slot < 0 || slot >= a.pool_rows ||
                       (a.freqs && !has_freq_row(pos, a.ratio, a.freq_rows));
  f32x4 fa = {1.f, 0.f, 1.f, 0.f}, fb = fa;
  const bool rotated = a.freqs && j >= 8;
  if (rotated && !refused) {
    const float* const f = freq_row(a.freqs, pos, a.ratio) + 8 * (j - 8);
    fa = *(const f32x4*)f;
    fb = *(const f32x4*)(f + 4);
  }
  float sum = v[0] * v[0];
#pragma unroll
  for (int c = 1; c < 8; ++c) {
    const float sq = v[c] * v[c];
    sum = sum + sq;
  }
  sum = sum + dpp<kXor1>(sum);
  sum = sum + dpp<kXor2>(sum);
  sum = sum + dpp<kHalfMirror>(sum);
  sum = sum + dpp<kMirror>(sum);
  const float r = inv_root(sum * (1.0f / kIndexDim) + a.eps);
  uint32_t n[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float lo = v[2 * c] * r, hi = v[2 * c + 1] * r;
    lo = lo * (c < 2 ? w0[2 * c] : w1[2 * c - 4]);
    hi = hi * (c < 2 ? w0[2 * c + 1] : w1[2 * c - 3]);
    n[c] = __builtin_bit_cast(uint32_t, bf16_pair(lo, hi));
  }
  if (rotated) {
    const float cs[8] = {fa[0], fa[1], fa[2], fa[3], fb[0], fb[1], fb[2], fb[3]};
    float nf[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      nf[2 * c] = u2f(n[c] << 16);
      nf[2 * c + 1] = u2f(n[c] & 0xffff0000u);
    }
    rope4(nf, cs);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      n[c] = __builtin_bit_cast(uint32_t, bf16_pair(nf[2 * c], nf[2 * c + 1]));
  }
  const uint32_t both = top_of_pairs(top_of_pairs(n[0], n[1]), top_of_pairs(n[2], n[3]));
  int top = (int)max(both & 0xffffu, both >> 16);
  top = max(top, dpp<kXor1>(top));
  top = max(top, dpp<kXor2>(top));
  top = max(top, dpp<kHalfMirror>(top));
  top = max(top, dpp<kMirror>(top));
  const bool special = top >= 0x7f80;  // an infinity or NaN in the row
  const float scale = exp2i(ue8m0_exponent(bf16_to_f32((uint32_t)top)));
  u32x2 code = {index_codes(n[0], n[1], scale), index_codes(n[2], n[3], scale)};
  if (special) code = u32x2{0, 0};
  if (refused) return;
  uint8_t* const page = a.pool + (int64_t)(slot >> 6) * kIndexPageBytes;
  *(u32x2*)(page + (slot & 63) * kIndexDim + 8 * j) = code;
  if (j == 0) *(float*)(page + kIndexScalesAt + 4 * (slot & 63)) = special ? NAN : scale;
}

struct GatherArgs {
  const uint8_t* pool;
  int64_t pool_rows;
  const int32_t* slots;
  int64_t stride_q, stride_k;
  const int32_t* lengths;
  int64_t length_stride;
  int64_t rows, k;
  uint16_t* out;
};
constexpr int kTurns = 4;  // of four rows, asked for together

__global__ __launch_bounds__(64 * kWaves) void index_gather_kernel(GatherArgs a) {
  const int lane = wave_lane(), j = lane & 15;
  const int64_t step = (int64_t)gridDim.x * kWaves * kTurns * 4;
  for (int64_t r0 = ((int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6)) * (kTurns * 4) + (lane >> 4);
       r0 < a.rows; r0 += step) {
    int32_t slot[kTurns];
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int64_t r = r0 + 4 * t;
      slot[t] = -1;
      if (r < a.rows) {
        const int64_t q = (uint32_t)r / (uint32_t)a.k;
        const int64_t k = r - q * a.k;
        const int64_t live = a.lengths ? a.lengths[q * a.length_stride] : a.k;
        if (k < live) slot[t] = a.slots[q * a.stride_q + k * a.stride_k];
        if (slot[t] >= a.pool_rows) slot[t] = -1;
      }
    }
    u32x2 code[kTurns];
    float scale[kTurns];
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      code[t] = u32x2{0, 0};
      scale[t] = 0.0f;
      if (slot[t] >= 0) {
        const uint8_t* const page = a.pool + (int64_t)(slot[t] >> 6) * kIndexPageBytes;
        code[t] = *(const u32x2*)(page + (slot[t] & 63) * kIndexDim + 8 * j);
        scale[t] = *(const float*)(page + kIndexScalesAt + 4 * (slot[t] & 63));
      }
    }
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      u32x4 o;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[t][c], false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[t][c], true);
        o[2 * c] = __builtin_bit_cast(uint32_t, bf16_pair(lo[0] * scale[t], lo[1] * scale[t]));
        o[2 * c + 1] = __builtin_bit_cast(uint32_t, bf16_pair(hi[0] * scale[t], hi[1] * scale[t]));
      }
      if (r0 + 4 * t < a.rows)
        __builtin_nontemporal_store(o, (u32x4*)(a.out + (r0 + 4 * t) * kIndexDim + 8 * j));
    }
  }
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

}  // namespace

extern "C" int rm_index_store_rows(const void* x, int x_dtype, int64_t x_row_stride,
                                   const float* weight, float eps, const int32_t* dst_slot,
                                   const int32_t* position, const float* freqs, int64_t freq_rows,
                                   int64_t ratio, int64_t n, uint8_t* pool, int64_t pool_pages,
                                   void* stream) {
  if (n < 0 || pool_pages < 0 || pool_pages > ((int64_t)1 << 25) || freq_rows < 0 || ratio < 1 ||
      ratio > 0x7fffffff || n > ((int64_t)1 << 34))
    return RM_ERR_SHAPE;
  if (n == 0) return RM_OK;
  if (!x || !weight || !dst_slot || !pool || (freqs && !position)) return RM_ERR_NULL;
  if (x_dtype != RM_F32 && x_dtype != RM_BF16) return RM_ERR_DTYPE;
  if (x_row_stride < kIndexDim && n > 1) return RM_ERR_SHAPE;
  if (!aligned(x, 16) || ((x_row_stride * (x_dtype == RM_BF16 ? 2 : 4)) & 15) ||
      !aligned(pool, 16) || !aligned(weight, 16) || !aligned(freqs, 16) || !aligned(dst_slot, 4) ||
      !aligned(position, 4))
    return RM_ERR_ALIGN;
  const int64_t row_bytes = x_row_stride * (x_dtype == RM_BF16 ? 2 : 4);
  for (int64_t at = 0; at < n; at += kLaunchRows) {
    const int64_t rows = std::min(n - at, kLaunchRows);
    const StoreArgs a{(const uint8_t*)x + at * row_bytes, x_row_stride, weight, eps, dst_slot + at,
                      freqs ? position + at : nullptr, freqs, freq_rows, rows, pool,
                      pool_pages * kPageRecords, (uint32_t)ratio};
    const unsigned blocks = (unsigned)((rows + 4 * kWaves - 1) / (4 * kWaves));
    hipLaunchKernelGGL(x_dtype == RM_BF16 ? index_store_kernel<true> : index_store_kernel<false>,
                       dim3(blocks), dim3(64 * kWaves), 0, (hipStream_t)stream, a);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  return RM_OK;
}

extern "C" int rm_index_gather_bf16(const uint8_t* pool, int64_t pool_pages, const int32_t* slots,
                                    int64_t slots_stride_q, int64_t slots_stride_k,
                                    const int32_t* lengths, int64_t length_stride,
                                    int64_t n_queries, int64_t selected_k, uint16_t* out,
                                    void* stream) {
  if (n_queries < 0 || selected_k < 0 || pool_pages < 0 || pool_pages > ((int64_t)1 << 25))
    return RM_ERR_SHAPE;
  if (selected_k > 0 && n_queries > 0xffffffffll / selected_k) return RM_ERR_SHAPE;
  if (n_queries == 0 || selected_k == 0) return RM_OK;
  if (!pool || !slots || !out) return RM_ERR_NULL;
  if (!aligned(pool, 16) || !aligned(out, 16) || !aligned(slots, 4) || !aligned(lengths, 4))
    return RM_ERR_ALIGN;
  const GatherArgs a{pool, pool_pages * kPageRecords, slots, slots_stride_q, slots_stride_k,
                     lengths, length_stride, n_queries * selected_k, selected_k, out};
  const int64_t blocks = (a.rows + 4 * kTurns * kWaves - 1) / (4 * kTurns * kWaves);
  hipLaunchKernelGGL(index_gather_kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)),
                     dim3(64 * kWaves), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
