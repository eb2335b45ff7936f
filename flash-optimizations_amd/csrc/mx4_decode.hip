// Sparse-MLA decode over 4-bit records, jointly with sliding-window rows of a
// Native pool. For query token t and head h, over the valid entries j of t's list
// and window (K_j the dequantized 512-coordinate row, V = K):
//   l_j = (q_h . K_j) * scale, Z = sum_j exp(l_j) + exp(sink_h),
//   out = sum_j exp(l_j) K_j / Z, lse = ln Z.
//
// One workgroup a (token, head); each wave takes every fourth entry, lane l the
// coordinates 8l..8l+7, with a running maximum and sum; the waves' parts meet in
// LDS.
#include "mx4_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kMaxTopk = 1 << 20;
constexpr int kMaxWindow = 512;
constexpr int kMaxHeads = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_len, heads;
  const uint8_t* pool;
  int64_t pool_pages;
  const int32_t* block_table;
  int64_t bt_stride, max_blocks;
  const int32_t* seqlens;
  const int32_t* indices;
  int64_t topk;
  const int32_t* topk_length;
  const uint8_t* swa_pool;
  int64_t swa_rows;
  const int32_t* swa_indices;
  int64_t swa_topk;
  const int32_t* swa_length;
  const float* sink;
  float scale_log2;
  uint16_t* out;
  float* lse;
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
  return x;
}

__global__ __launch_bounds__(256) void mx4_decode_kernel(DecodeArgs a) {
  __shared__ float part_o[4][kHeadDim], part_m[4], part_l[4];
  const int lane = wave_lane();
  const int wave = uniform((int)(threadIdx.x >> 6));
  const int64_t t = blockIdx.y, h = blockIdx.x, request = t / a.q_len;
  float q[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = bf16_to_f32(a.q[(t * a.heads + h) * kHeadDim + 8 * lane + i]);
    o[i] = 0.0f;
  }
  auto take = [&](const u32x4& row) {
    float k[8], s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      k[i] = bf16_to_f32((row[i / 2] >> (16 * (i % 2))) & 0xffffu);
      s += q[i] * k[i];
    }
    s = wave_sum(s) * a.scale_log2;
    const float mn = fmaxf(m, s);
    const float f = exp2f(m - mn), p = exp2f(s - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * f + p * k[i];
    m = mn;
  };
  int64_t live = a.topk;
  if (a.topk_length) live = min((int64_t)a.topk_length[t], live);
  const int64_t records = a.seqlens ? a.seqlens[request] : (int64_t)1 << 40;
  for (int64_t j = wave; j < live; j += 4) {
    const int64_t r = a.indices[t * a.topk + j];
    if (r < 0 || r >= records || r / kPageRecords >= a.max_blocks) continue;
    const int64_t page = a.block_table[request * a.bt_stride + r / kPageRecords];
    if (page < 0 || page >= a.pool_pages) continue;
    const uint8_t* rec = a.pool + (page * kPageRecords + r % kPageRecords) * kMx4RecordBytes;
    take(fp4x8_to_bf16(*(const uint32_t*)(rec + 4 * lane),
                       mx4_scale(rec[kMx4CodeBytes + (lane >> 2)])));
  }
  int64_t window = a.swa_topk;
  if (a.swa_length) window = min((int64_t)a.swa_length[t], window);
  for (int64_t j = wave; j < window; j += 4) {
    const int64_t slot = a.swa_indices[t * a.swa_topk + j];
    if (slot < 0 || slot >= a.swa_rows) continue;
    const uint8_t* page = a.swa_pool + slot / kPageRecords * kNativePageBytes;
    const int row = (int)(slot % kPageRecords);
    const uint8_t* data = page + row * kNativeDataBytes;
    u32x4 v;
    if (lane < kNopeDim / 8) {
      const u32x2 codes = *(const u32x2*)(data + 8 * lane);
      const float scale = u2f((uint32_t)page[kPageRecords * kNativeDataBytes + row * kScaleBytes +
                                             (lane >> 3)] << 23);
      v = u32x4{fp8_pair_to_bf16<false>(codes[0], scale), fp8_pair_to_bf16<true>(codes[0], scale),
                fp8_pair_to_bf16<false>(codes[1], scale), fp8_pair_to_bf16<true>(codes[1], scale)};
    } else {
      v = *(const u32x4*)(data + kNopeDim + 16 * (lane - kNopeDim / 8));
    }
    take(v);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part_o[wave][8 * lane + i] = o[i];
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
  __syncthreads();
  const float sink = a.sink ? a.sink[h] * kLog2e : -INFINITY;
  float top = sink;
  for (int w = 0; w < 4; ++w) top = part_l[w] == 0.0f ? top : fmaxf(top, part_m[w]);
  float z = 0.0f, f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = part_l[w] == 0.0f ? 0.0f : exp2f(part_m[w] - top);
    z += f[w] * part_l[w];
  }
  if (top != -INFINITY) z += exp2f(sink - top);
  const float inv = z != 0.0f ? 1.0f / z : 0.0f;
  for (int c = threadIdx.x; c < kHeadDim; c += 256) {
    float v = 0.0f;
    for (int w = 0; w < 4; ++w)
      if (f[w] != 0.0f) v += f[w] * part_o[w][c];
    a.out[(t * a.heads + h) * kHeadDim + c] = __builtin_bit_cast(uint16_t, (__bf16)(v * inv));
  }
  if (threadIdx.x == 0) a.lse[t * a.heads + h] = z != 0.0f ? (top + log2f(z)) * kLn2 : -INFINITY;
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

bool bad_sizes(int64_t tokens, int64_t heads, int64_t topk, int64_t swa_topk) {
  return tokens < 0 || tokens > 65535 || heads < 0 || heads > kMaxHeads || topk < 0 ||
         topk > kMaxTopk || swa_topk < 0 || swa_topk > kMaxWindow;
}

}  // namespace

extern "C" int rm_mx4_sparse_decode_workspace(int64_t tokens, int64_t heads, int64_t topk,
                                              int64_t swa_topk, int32_t* num_splits,
                                              size_t* workspace_bytes) {
  if (bad_sizes(tokens, heads, topk, swa_topk)) return RM_ERR_SHAPE;
  if (num_splits) *num_splits = 1;
  if (workspace_bytes) *workspace_bytes = 0;
  return RM_OK;
}

extern "C" int rm_mx4_sparse_decode_fwd(
    const uint16_t* q, int64_t batch, int64_t q_len, int64_t heads, const uint8_t* pool,
    int64_t pool_pages, const int32_t* block_table, int64_t block_table_stride,
    int64_t max_blocks, const int32_t* seqlens, const int32_t* indices, int64_t topk,
    const int32_t* topk_length, const uint8_t* swa_pool, int64_t swa_pool_pages,
    const int32_t* swa_indices, int64_t swa_topk, const int32_t* swa_length, const float* sink,
    float softmax_scale, uint16_t* out, float* lse, void* workspace, size_t workspace_bytes,
    void* stream) {
  if (batch < 0 || q_len < 0 || batch > 65535 || q_len > 65535 ||
      bad_sizes(batch * q_len, heads, topk, swa_topk) || pool_pages < 0 || max_blocks < 0 ||
      max_blocks > 0x7fffffff || swa_pool_pages < 0 || pool_pages > ((int64_t)1 << 25) ||
      swa_pool_pages > ((int64_t)1 << 25) || block_table_stride < max_blocks)
    return RM_ERR_SHAPE;
  const int64_t tokens = batch * q_len;
  if (tokens == 0 || heads == 0) return RM_OK;
  if (!q || !out || !lse || (topk > 0 && (!indices || !pool || !block_table)) ||
      (swa_topk > 0 && (!swa_indices || !swa_pool)))
    return RM_ERR_NULL;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(pool, 16) ||
      !aligned(swa_pool, 16))
    return RM_ERR_ALIGN;
  const DecodeArgs a{q, q_len, heads, pool, pool_pages, block_table, block_table_stride,
                     max_blocks, seqlens, indices, topk, topk_length, swa_pool,
                     swa_pool_pages * kPageRecords, swa_indices, swa_topk, swa_length, sink,
                     softmax_scale * kLog2e, out, lse};
  hipLaunchKernelGGL(mx4_decode_kernel, dim3((unsigned)heads, (unsigned)tokens), dim3(256), 0,
                     (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
