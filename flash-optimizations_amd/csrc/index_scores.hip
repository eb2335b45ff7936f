// Scores of cached index records: for query token t with H heads q_h (BF16) and head
// weights w, record r of its request,
//   s[t, r] = c_r * sum_h (w_h c_h) max(0, sum_d Q8_h[d] K8_r[d]),
// where Q8_h, c_h are q_h coded as the store codes a key (codes and a power of two a row
// of 128) and K8_r, c_r the cached record. -inf where r is past the token's length or its
// page is not mapped.
//
// Codes are multiplied as BF16, which holds them: v_mfma_f32_16x16x32_bf16 adds their
// products as float32 does, while this card's 8-bit matrix instructions (both
// 16x16x32 and 16x16x128, at the same and twice the rate) were 4e-5 of the result off on
// codes of eight octaves. A wave holds its tokens' coded heads in registers as first
// operands, 16 heads a tile, and takes its pages in turn, 16 records a tile as second
// operands, converted once for all of its tokens. (Which coordinate stands where in the
// long axis is free as long as both operands agree: a lane takes coordinates 16 g .. + 15 and
// 64 + 16 g .. + 15 of its row, two 16-byte loads of a record that together use whole
// 64-byte pieces.) The products come out with a lane's four heads of one record beside
// each other, so the weighted sum over heads is in the lane; the four lanes of a record
// meet once a page, where record l of the page ends in lane l and its scale, score
// and store are one access a wave.
#include <algorithm>

#include "index_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kWaves = 4;

struct ScoreArgs {
  const uint16_t* q;     // [batch, q_len, heads, 128]
  const float* weights;  // [batch, q_len, heads]
  int q_len, heads;
  const uint8_t* pool;
  int pool_pages;
  const int32_t* block_table;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* lengths;  // [batch * q_len]
  int64_t width;
  float* out;  // [batch * q_len, width]
  int pages;   // of a row of out
  int groups;  // workgroups along the tokens of a request
};

__device__ __forceinline__ uint32_t over_groups_top(uint32_t x) {
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(b[0], b[1]);
}
// Eight codes -> eight BF16.
__device__ __forceinline__ bf16x8 values_of(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(
      bf16x8, u32x4{fp8_pair_to_bf16<false>(lo, 1.0f), fp8_pair_to_bf16<true>(lo, 1.0f),
                    fp8_pair_to_bf16<false>(hi, 1.0f), fp8_pair_to_bf16<true>(hi, 1.0f)});
}

// kTiles x 16 heads, kTokens tokens a wave. kApart: the waves of a workgroup take
// different tokens and the same pages; otherwise the same tokens and pages in turn.
template <int kTiles, int kTokens, bool kApart>
__global__ __launch_bounds__(64 * kWaves) void index_scores_kernel(ScoreArgs a) {
  const int lane = wave_lane(), row = lane & 15, group = lane >> 4;
  const int wave = uniform((int)(threadIdx.x >> 6));
  const int b = (int)blockIdx.x / a.groups;
  const int of = (int)blockIdx.x - b * a.groups;
  const int t0 = of * kTokens * (kApart ? kWaves : 1) + (kApart ? wave * kTokens : 0);
  if (t0 >= a.q_len) return;
  const int64_t first = (int64_t)b * a.q_len + t0;  // row of q, lengths and out
  const int32_t* const table = a.block_table + b * a.bt_stride;
  int length[kTokens], most = 0;
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    length[t] = 0;
    if (t0 + t < a.q_len)
      length[t] = (int)min((int64_t)max(a.lengths[first + t], 0),
                           min(a.width, (int64_t)a.max_blocks * kPageRecords));
    most = max(most, length[t]);
  }
  const int live = (most + kPageRecords - 1) / kPageRecords;  // pages to score
  const int step = (int)gridDim.y * (kApart ? 1 : kWaves);
  int p = kApart ? (int)blockIdx.y : (int)blockIdx.y * kWaves + wave;

  bf16x8 q[kTokens][kTiles][4];
  f32x4 w[kTokens][kTiles];
  if (p < live) {
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const int h = 16 * i + row;
        u32x4 x[4] = {};
        float weight = 0.0f;
        if (t0 + t < a.q_len && h < a.heads) {
          const int64_t at = (first + t) * a.heads + h;
          const u32x4* const from = (const u32x4*)(a.q + at * kIndexDim);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] = from[2 * group + (k & 1) + 8 * (k >> 1)];
          weight = a.weights[at];
        }
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          top = top_of_pairs(top, top_of_pairs(top_of_pairs(x[k][0], x[k][1]),
                                               top_of_pairs(x[k][2], x[k][3])));
        top = over_groups_top(max(top & 0xffffu, top >> 16));
        const bool special = top >= 0x7f80u;  // an infinity or NaN in the row
        const float scale = exp2i(ue8m0_exponent(bf16_to_f32(top)));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t lo = index_codes(x[k][0], x[k][1], scale);
          const uint32_t hi = index_codes(x[k][2], x[k][3], scale);
          q[t][i][k] = values_of(special ? 0u : lo, special ? 0u : hi);
        }
        // the product's rows 4 group + c of a tile: those heads' weights
        const float all = special ? NAN : weight * scale;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          w[t][i][c] = u2f((uint32_t)__builtin_amdgcn_ds_bpermute(4 * (4 * group + c),
                                                                  (int)f2u(all)));
      }
    }
  }
  for (; p < a.pages; p += step) {
    const int64_t r = (int64_t)p * kPageRecords + lane;
    float s[kTokens];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) s[t] = -INFINITY;
    const int page = p < live ? table[p] : -1;
    if (page >= 0 && page < a.pool_pages) {
      const uint8_t* const from = a.pool + (int64_t)page * kIndexPageBytes;
      const float scale = *(const float*)(from + kIndexScalesAt + 4 * lane);
      u32x4 raw[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4* const at = (const u32x4*)(from + (16 * i + row) * kIndexDim) + group;
        raw[i][0] = at[0];
        raw[i][1] = at[4];
      }
      float sum[kTokens][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bf16x8 k[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          k[n] = values_of(raw[i][n / 2][2 * (n & 1)], raw[i][n / 2][2 * (n & 1) + 1]);
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
          f32x4 d[kTiles];
#pragma unroll
          for (int h = 0; h < kTiles; ++h) d[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int h = 0; h < kTiles; ++h)
              d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q[t][h][n], k[n], d[h], 0, 0, 0);
          float all = 0.0f;
#pragma unroll
          for (int h = 0; h < kTiles; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c)  // (a NaN stays one)
              all = __builtin_fmaf(w[t][h][c], __builtin_elementwise_maximum(d[h][c], 0.0f), all);
          sum[t][i] = all;
        }
      }
#pragma unroll
      for (int t = 0; t < kTokens; ++t) {
        // over the four lanes of a record; lane l ends with record l
        const auto x02 = __builtin_amdgcn_permlane32_swap(f2u(sum[t][0]), f2u(sum[t][2]), false, false);
        const auto x13 = __builtin_amdgcn_permlane32_swap(f2u(sum[t][1]), f2u(sum[t][3]), false, false);
        const float lo = u2f(x02[0]) + u2f(x02[1]), hi = u2f(x13[0]) + u2f(x13[1]);
        const auto x = __builtin_amdgcn_permlane16_swap(f2u(lo), f2u(hi), false, false);
        if (r < length[t]) s[t] = scale * (u2f(x[0]) + u2f(x[1]));
      }
    }
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
      if (t0 + t < a.q_len && r < a.width) a.out[(first + t) * a.width + r] = s[t];
  }
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

}  // namespace

extern "C" int rm_index_scores(const uint16_t* q, int64_t batch, int64_t q_len, int64_t heads,
                               const float* weights, const uint8_t* pool, int64_t pool_pages,
                               const int32_t* block_table, int64_t block_table_stride,
                               int64_t max_blocks, const int32_t* lengths, int64_t width,
                               float* out, void* stream) {
  if (batch < 0 || q_len < 0 || heads < 0 || heads > RM_MAX_INDEX_HEADS || batch > 65535 ||
      q_len > (1 << 20) || batch * q_len > (1 << 20) || pool_pages < 0 ||
      pool_pages > ((int64_t)1 << 25) || max_blocks < 0 || max_blocks > ((int64_t)1 << 25) ||
      block_table_stride < max_blocks || width < 0 || width > 0x7fffffff - 64)
    return RM_ERR_SHAPE;
  if (batch == 0 || q_len == 0 || width == 0) return RM_OK;
  if (!lengths || !out || (heads > 0 && (!q || !weights)) ||
      (max_blocks > 0 && (!block_table || (pool_pages > 0 && !pool))))
    return RM_ERR_NULL;
  if (!aligned(q, 16) || !aligned(pool, 16) || !aligned(weights, 4) || !aligned(block_table, 4) ||
      !aligned(lengths, 4) || !aligned(out, 4))
    return RM_ERR_ALIGN;
  ScoreArgs a{q, weights, (int)q_len, (int)heads, pool, (int)pool_pages, block_table,
              block_table_stride, (int)max_blocks, lengths, width, out,
              (int)((width + kPageRecords - 1) / kPageRecords), 0};
  const int tokens = q_len > 1 && heads <= 64 ? 2 : 1;
  const bool apart = q_len >= 8 * kWaves;
  a.groups = (int)((q_len + tokens * (apart ? kWaves : 1) - 1) / (tokens * (apart ? kWaves : 1)));
  const int64_t rows = batch * a.groups;
  const int64_t turns = (a.pages + (apart ? 1 : kWaves) - 1) / (apart ? 1 : kWaves);
  const int64_t splits = std::min<int64_t>(turns, std::max<int64_t>(1, 2048 / rows));
  const auto pick = [&](auto one, auto two, auto more) { return apart ? more : tokens == 2 ? two : one; };
  const auto kern =
      heads <= 16   ? pick(index_scores_kernel<1, 1, false>, index_scores_kernel<1, 2, false>, index_scores_kernel<1, 2, true>)
      : heads <= 32 ? pick(index_scores_kernel<2, 1, false>, index_scores_kernel<2, 2, false>, index_scores_kernel<2, 2, true>)
      : heads <= 64 ? pick(index_scores_kernel<4, 1, false>, index_scores_kernel<4, 2, false>, index_scores_kernel<4, 2, true>)
                    : pick(index_scores_kernel<8, 1, false>, index_scores_kernel<8, 1, false>, index_scores_kernel<8, 1, true>);
  hipLaunchKernelGGL(kern, dim3((unsigned)rows, (unsigned)splits), dim3(64 * kWaves), 0,
                     (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
