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
// operands, 16 heads a tile, and takes pages in turn, 16 records a tile as second
// operands, converted once for all of its tokens. (Which coordinate stands where in the
// long axis is free as long as both operands agree: a lane takes coordinates 16 g .. + 15 and
// 64 + 16 g .. + 15 of its row, two 16-byte loads of a record that together use whole
// 64-byte pieces.) A tile's registers take the next page's records as soon as they are
// converted, so a page is in flight while one is multiplied. The products come out with a
// lane's four heads of one record beside each other, so the weighted sum over heads is in
// the lane; the four lanes of a record meet once a page, where record l of the page ends in
// lane l and its scale, score and store are one access a wave.
//
// Bound by the products for many tokens (512 tokens, 35,840 records: 231 us, 1,310 TFLOP/s; a
// large library product reaches 1,189), by the matrix instructions and by memory alike for
// two tokens of 64 heads (128 requests of 32,768 records: 145 us; 108 for the bytes at 5.1 TB/s,
// 105 for the products at 1,310 TFLOP/s), by memory and its latency for one (64 ragged
// requests 24 us, 17 for the bytes).
#include <algorithm>

#include "index_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kWaves = 4;

typedef __attribute__((address_space(4))) int32_t const_i32;  // scalar loads

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
  int least;   // pages that a wave takes at least, if there are
  int splits;  // workgroups of a row of them
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

// A tile of heads as the products take it: coordinates 64 (k / 2) + 16 group + 8 (k % 2) ..
// of head `row` in x[k], and its weight times its scale (NaN for a row with an infinity or
// NaN, whose codes are zeros).
struct Heads {
  bf16x8 x[4];
  float weight;
};
__device__ __forceinline__ Heads coded(const ScoreArgs& a, int64_t token, int h, int group) {
  u32x4 x[4] = {};
  float weight = 0.0f;
  if (h < a.heads) {
    const int64_t at = token * a.heads + h;
    const u32x4* const from = (const u32x4*)(a.q + at * kIndexDim);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = from[2 * group + (k & 1) + 8 * (k >> 1)];
    weight = a.weights[at];
  }
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    top = top_of_pairs(top,
                       top_of_pairs(top_of_pairs(x[k][0], x[k][1]), top_of_pairs(x[k][2], x[k][3])));
  top = over_groups_top(max(top & 0xffffu, top >> 16));
  const bool special = top >= 0x7f80u;
  const float scale = exp2i(ue8m0_exponent(bf16_to_f32(top)));
  Heads to;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = index_codes(x[k][0], x[k][1], scale);
    const uint32_t hi = index_codes(x[k][2], x[k][3], scale);
    to.x[k] = values_of(special ? 0u : lo, special ? 0u : hi);
  }
  to.weight = special ? NAN : weight * scale;
  return to;
}

// kTiles x 16 heads, kTokens tokens a wave. kApart: the waves of a workgroup take
// different tokens and the same pages; otherwise the same tokens and pages in turn, and
// each codes some of the heads for all.
constexpr int waves_a_simd(int tiles, int tokens) {
  return tiles * tokens >= 8 ? 2 : tiles >= 4 ? 3 : tokens >= 2 ? 2 : 4;
}
template <int kTiles, int kTokens, bool kApart>
__global__ __launch_bounds__(64 * kWaves, waves_a_simd(kTiles, kTokens)) void index_scores_kernel(
    ScoreArgs a) {
  constexpr int kShared = kApart ? 1 : kTokens * kTiles;
  __shared__ u32x4 coded_heads[kShared][4][64];
  // (weights stay there: 2 x 64 heads and theirs in registers would spill)
  __shared__ f32x4 head_weights[kApart ? kWaves : 1][kTokens * kTiles][4];
  const int lane = wave_lane(), row = lane & 15, group = lane >> 4;
  const int wave = uniform((int)(threadIdx.x >> 6));
  const int row_of_groups = (int)(blockIdx.x / (uint32_t)a.splits);
  const int split = (int)blockIdx.x - row_of_groups * a.splits;
  const int b = row_of_groups / a.groups;
  const int of = row_of_groups - b * a.groups;
  const int t0 = of * kTokens * (kApart ? kWaves : 1) + (kApart ? wave * kTokens : 0);
  if (t0 >= a.q_len) return;
  const int64_t first = (int64_t)b * a.q_len + t0;  // row of q, lengths and out
  const const_i32* const table = (const const_i32*)a.block_table + b * a.bt_stride;
  int length[kTokens], most = 0;
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    length[t] = 0;
    if (t0 + t < a.q_len)
      length[t] = (int)min((int64_t)max(((const const_i32*)a.lengths)[first + t], 0),
                           min(a.width, (int64_t)a.max_blocks * kPageRecords));
    most = max(most, length[t]);
  }
  const int live = (most + kPageRecords - 1) / kPageRecords;  // pages to score
  // of `of_all` waves (workgroups) that take pages in turn, `working` have scores to find
  const int of_all = a.splits * (kApart ? 1 : kWaves);
  const int turn = (split + row_of_groups) % a.splits;
  const int start = kApart ? turn : turn * kWaves;
  const int me = start + (kApart ? 0 : wave);
  int working = of_all;
  if (!kApart)
    working = min(of_all, ((live + a.least - 1) / a.least + kWaves - 1) / kWaves * kWaves);
  auto put = [&](int p, const float (&s)[kTokens]) {
    const int64_t r = (int64_t)p * kPageRecords + lane;
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
      if (t0 + t < a.q_len && r < a.width) a.out[(first + t) * a.width + r] = s[t];
  };
  float none[kTokens];
#pragma unroll
  for (int t = 0; t < kTokens; ++t) none[t] = -INFINITY;
  for (int p = live + me; p < a.pages; p += of_all) put(p, none);
  if (start >= min(live, working)) return;

  constexpr int kAll = kTokens * kTiles, kAtOnce = kAll < 4 ? kAll : 4;
  bf16x8 q[kAll][4];  // tile i of token t: kTiles t + i
  if constexpr (kApart) {
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const Heads x = coded(a, first + t, t0 + t < a.q_len ? 16 * i + row : a.heads, group);
#pragma unroll
        for (int k = 0; k < 4; ++k) q[kTiles * t + i][k] = x.x[k];
        if (group == 0) ((float*)&head_weights[wave][kTiles * t + i][0])[row] = x.weight;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
#pragma unroll 1
    for (int n = 0; n < kShared; n += kWaves) {
      const int at = n + wave, t = at / kTiles, i = at - t * kTiles;
      if (kShared % kWaves == 0 || at < kShared) {
        const Heads x = coded(a, first + t, t0 + t < a.q_len ? 16 * i + row : a.heads, group);
#pragma unroll
        for (int k = 0; k < 4; ++k) coded_heads[at][k][lane] = __builtin_bit_cast(u32x4, x.x[k]);
        if (group == 0) ((float*)&head_weights[0][at][0])[row] = x.weight;
      }
    }
    __syncthreads();
    if (me >= min(live, working)) return;
#pragma unroll
    for (int i = 0; i < kAll; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) q[i][k] = __builtin_bit_cast(bf16x8, coded_heads[i][k][lane]);
    }
  }
  // Records 16 i + row of a page, and the scale of record lane. (A page that is not mapped:
  // page 0's, which nobody looks at.)
  u32x4 raw[4][2];
  float scale;
  auto mapped = [&](int page) { return page >= 0 && page < a.pool_pages; };
  auto base = [&](int page) {
    return a.pool + (int64_t)(mapped(page) ? page : 0) * kIndexPageBytes;
  };
  auto fetch = [&](const uint8_t* from, int i) {
    const u32x4* const at = (const u32x4*)(from + (16 * i + row) * kIndexDim) + group;
    raw[i][0] = at[0];
    raw[i][1] = at[4];
  };
  int page = table[me];
  int next = me + working < live ? table[me + working] : -1;
  {
    const uint8_t* const from = base(page);
#pragma unroll
    for (int i = 0; i < 4; ++i) fetch(from, i);
    scale = *(const float*)(from + kIndexScalesAt + 4 * lane);
  }
  for (int p = me; p < live; p += working) {
    const int after = p + 2 * working < live ? table[p + 2 * working] : -1;
    const uint8_t* const ahead = base(next);  // (once past the end: page 0 again)
    // the product's rows 4 group + c of a tile: those heads' weights
    int of_group = group;
    asm volatile("" : "+v"(of_group));
    float sum[kTokens][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x8 k[4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
        k[n] = values_of(raw[i][n / 2][2 * (n & 1)], raw[i][n / 2][2 * (n & 1) + 1]);
      fetch(ahead, i);
#pragma unroll
      for (int t = 0; t < kTokens; ++t) sum[t][i] = 0.0f;
#pragma unroll
      for (int from = 0; from < kAll; from += kAtOnce) {
        f32x4 d[kAtOnce];
#pragma unroll
        for (int h = 0; h < kAtOnce; ++h) d[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int h = 0; h < kAtOnce; ++h)
            d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q[from + h][n], k[n], d[h], 0, 0, 0);
#pragma unroll
        for (int h = 0; h < kAtOnce; ++h) {
          float& all = sum[(from + h) / kTiles][i];
          const f32x4 w = head_weights[kApart ? wave : 0][from + h][of_group];
#pragma unroll
          for (int c = 0; c < 4; ++c)  // (a NaN stays one)
            all = __builtin_fmaf(w[c], __builtin_elementwise_maximum(d[h][c], 0.0f), all);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    float s[kTokens];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      // over the four lanes of a record; lane l ends with record l
      const auto x02 = __builtin_amdgcn_permlane32_swap(f2u(sum[t][0]), f2u(sum[t][2]), false, false);
      const auto x13 = __builtin_amdgcn_permlane32_swap(f2u(sum[t][1]), f2u(sum[t][3]), false, false);
      const float lo = u2f(x02[0]) + u2f(x02[1]), hi = u2f(x13[0]) + u2f(x13[1]);
      const auto x = __builtin_amdgcn_permlane16_swap(f2u(lo), f2u(hi), false, false);
      s[t] = scale * (u2f(x[0]) + u2f(x[1]));
      if (!mapped(page) || p * kPageRecords + lane >= length[t]) s[t] = -INFINITY;
    }
    scale = *(const float*)(ahead + kIndexScalesAt + 4 * lane);
    put(p, s);
    page = next;
    next = after;
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
              block_table_stride, pool_pages > 0 ? (int)max_blocks : 0, lengths, width, out,
              (int)((width + kPageRecords - 1) / kPageRecords), 0, 1, 1};
  // Tokens of a wave: as many as make eight tiles of heads, as each page is converted for all
  // of them at once (3 x 257 tokens of 32 heads, 25,286 records: 156 us; 185 with two), or two
  // if there is not that much to do (4 tokens of 32 heads, 999 records: 5.7 us; 7.3 with four).
  const int tiles = heads <= 16 ? 1 : heads <= 32 ? 2 : heads <= 64 ? 4 : 8;
  const int full = 8 / tiles;
  const bool much = batch * q_len * a.pages >= 16384;
  const int tokens = q_len >= full && (much || full <= 2) ? full : q_len > 1 ? 2 : 1;
  const bool apart = q_len >= 8 * kWaves && tokens == full;
  a.groups = (int)((q_len + tokens * (apart ? kWaves : 1) - 1) / (tokens * (apart ? kWaves : 1)));
  const int64_t rows = batch * a.groups;
  const int64_t turns = (a.pages + (apart ? 1 : kWaves) - 1) / (apart ? 1 : kWaves);
  // Workgroups: two turns of what the chip holds, which is two waves a SIMD with 128 coded
  // heads in registers and three or more with fewer (64 ragged requests: 2,048 23.6 us,
  // 1,536 24.7, 1,024 28.9; 128 requests of 2 tokens: 1,024 145 us, 2,048 151, 512 142).
  // A wave takes four pages at least once there are that many, as its heads cost it about
  // as much as one (64 ragged requests, of two pages 26.9 us, of six 28.9), and where it codes
  // all of them itself as much as three (3 x 257 tokens, 333 records: 19.0 us; 25.4 of one).
  const int64_t most = tokens * tiles >= 8 ? 1024 : 2048;
  int64_t splits = std::min<int64_t>(turns, std::max<int64_t>(1, most / rows));
  a.least = (int)std::min<int64_t>(std::max<int64_t>(rows * a.pages / (apart ? 256 : 4096), 1), 4);
  if (apart) splits = std::min<int64_t>(splits, std::max<int64_t>(1, a.pages / a.least));
  a.splits = (int)splits;
  const auto pick = [&](auto one, auto two, auto more, auto many) {
    return apart ? many : tokens > 2 ? more : tokens == 2 ? two : one;
  };
  const auto kern =
      tiles == 1   ? pick(index_scores_kernel<1, 1, false>, index_scores_kernel<1, 2, false>,
                          index_scores_kernel<1, 8, false>, index_scores_kernel<1, 8, true>)
      : tiles == 2 ? pick(index_scores_kernel<2, 1, false>, index_scores_kernel<2, 2, false>,
                          index_scores_kernel<2, 4, false>, index_scores_kernel<2, 4, true>)
      : tiles == 4 ? pick(index_scores_kernel<4, 1, false>, index_scores_kernel<4, 2, false>,
                          index_scores_kernel<4, 2, false>, index_scores_kernel<4, 2, true>)
                   : pick(index_scores_kernel<8, 1, false>, index_scores_kernel<8, 1, false>,
                          index_scores_kernel<8, 1, false>, index_scores_kernel<8, 1, true>);
  hipLaunchKernelGGL(kern, dim3((unsigned)(splits * rows)), dim3(64 * kWaves), 0,
                     (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
