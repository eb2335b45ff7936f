// Reader of 4-bit records: row (q, k) of the output is record slots[q, k] as 512
// BF16 values (exact: a code times a power of two), zeros where the entry is
// padding or outside the pool.
//
// One wave a row; lane l expands the dword of coordinates 8l..8l+7 and writes them
// as one 16-byte piece, so a wave writes its 1 KiB row coalesced.
#include <algorithm>

#include "mx4_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kWaves = 4;

struct GatherArgs {
  const uint8_t* pool;
  int64_t pool_rows;
  const int32_t* slots;
  int64_t stride_q, stride_k;
  const int32_t* lengths;
  int64_t length_stride;
  int64_t queries, k;
  uint16_t* out;
};

__global__ __launch_bounds__(256) void mx4_gather_kernel(GatherArgs a) {
  const int lane = wave_lane();
  const int wave = uniform((int)(threadIdx.x >> 6));
  for (int64_t q = blockIdx.y; q < a.queries; q += gridDim.y) {
    const int64_t live = a.lengths ? a.lengths[q * a.length_stride] : a.k;
    for (int64_t k = (int64_t)blockIdx.x * kWaves + wave; k < a.k;
         k += (int64_t)gridDim.x * kWaves) {
      int64_t slot = -1;
      if (k < live) slot = a.slots[q * a.stride_q + k * a.stride_k];
      u32x4 v = {0, 0, 0, 0};
      if (slot >= 0 && slot < a.pool_rows) {
        const uint8_t* rec = a.pool + slot * kMx4RecordBytes;
        const uint32_t codes = *(const uint32_t*)(rec + 4 * lane);
        v = fp4x8_to_bf16(codes, mx4_scale(rec[kMx4CodeBytes + (lane >> 2)]));
      }
      *(u32x4*)(a.out + (q * a.k + k) * kHeadDim + 8 * lane) = v;
    }
  }
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

}  // namespace

extern "C" int rm_mx4_gather_bf16(const uint8_t* pool, int64_t pool_pages, const int32_t* slots,
                                  int64_t slots_stride_q, int64_t slots_stride_k,
                                  const int32_t* lengths, int64_t length_stride,
                                  int64_t n_queries, int64_t selected_k, uint16_t* out,
                                  void* stream) {
  if (n_queries < 0 || selected_k < 0 || pool_pages < 0 || pool_pages > ((int64_t)1 << 25))
    return RM_ERR_SHAPE;
  if (selected_k > 0 && n_queries > ((int64_t)1 << 40) / selected_k) return RM_ERR_SHAPE;
  if (n_queries == 0 || selected_k == 0) return RM_OK;
  if (!pool || !slots || !out) return RM_ERR_NULL;
  if (!aligned(pool, 16) || !aligned(out, 16) || !aligned(slots, 4) || !aligned(lengths, 4))
    return RM_ERR_ALIGN;
  const GatherArgs a{pool, pool_pages * kPageRecords, slots, slots_stride_q, slots_stride_k,
                     lengths, length_stride, n_queries, selected_k, out};
  const int64_t across = std::min<int64_t>((selected_k + kWaves - 1) / kWaves, 256 * 64);
  const dim3 grid((unsigned)across, (unsigned)std::min<int64_t>(n_queries, 65535));
  hipLaunchKernelGGL(mx4_gather_kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
