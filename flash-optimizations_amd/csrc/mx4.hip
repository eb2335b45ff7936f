// Reader of 4-bit records: row (q, k) of the output is record slots[q, k] as 512
// BF16 values (exact: a code times a power of two), zeros where the entry is
// padding or outside the pool.
//
// Four rows a wave, their records all asked for before the first is expanded; lane
// l expands the dword of coordinates 8l..8l+7 of each and writes them as one
// 16-byte piece, so a wave writes each 1 KiB row coalesced. Bound by memory: 272
// bytes read at random and 1,024 written for a row.
//
// 1,048,576 rows take 242 us (5.6 TB/s; a 1 GiB copy moves 5.1), 35,840 rows 9.7 us
// and 16 x 512 rows 3.9 us. One row a wave: 333 (plain stores: 328) / 11.0 / 4.1;
// two 249 / 9.7 / 3.8; eight 249 / 9.8 / 3.9; four with plain instead of
// non-temporal stores 276 / 10.5 / 4.3; sixteen in four turns 268 / 10.4 / 5.1.
#include <algorithm>

#include "mx4_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kWaves = 4;
constexpr int kRows = 4;  // rows a wave has in flight

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

__global__ __launch_bounds__(256) void mx4_gather_kernel(GatherArgs a) {
  const int lane = wave_lane();
  const int64_t step = (int64_t)gridDim.x * kWaves * kRows;
  for (int64_t r0 = ((int64_t)blockIdx.x * kWaves + uniform((int)(threadIdx.x >> 6))) * kRows;
       r0 < a.rows; r0 += step) {
    const int64_t r = r0 + lane;
    int32_t slot = -1;  // lane i: the slot of row r0 + i
    if (lane < kRows && r < a.rows) {
      const int64_t q = (uint32_t)r / (uint32_t)a.k;
      const int64_t k = r - q * a.k;
      const int64_t live = a.lengths ? a.lengths[q * a.length_stride] : a.k;
      if (k < live) slot = a.slots[q * a.stride_q + k * a.stride_k];
      if (slot >= a.pool_rows) slot = -1;
    }
    uint32_t codes[kRows], scale[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int32_t s = __builtin_amdgcn_readlane(slot, j);
      codes[j] = scale[j] = 0;
      if (s >= 0) {
        const uint8_t* const rec = a.pool + (int64_t)s * kMx4RecordBytes;
        codes[j] = *(const uint32_t*)(rec + 4 * lane);
        scale[j] = rec[kMx4CodeBytes + (lane >> 2)];
      }
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (r0 + j < a.rows)  // written once and larger than the caches as a rule
        __builtin_nontemporal_store(fp4x8_to_bf16(codes[j], mx4_scale(scale[j])),
                                    (u32x4*)(a.out + (r0 + j) * kHeadDim + 8 * lane));
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
  if (selected_k > 0 && n_queries > 0xffffffffll / selected_k) return RM_ERR_SHAPE;
  if (n_queries == 0 || selected_k == 0) return RM_OK;
  if (!pool || !slots || !out) return RM_ERR_NULL;
  if (!aligned(pool, 16) || !aligned(out, 16) || !aligned(slots, 4) || !aligned(lengths, 4))
    return RM_ERR_ALIGN;
  const GatherArgs a{pool, pool_pages * kPageRecords, slots, slots_stride_q, slots_stride_k,
                     lengths, length_stride, n_queries * selected_k, selected_k, out};
  const int64_t blocks = (a.rows + kWaves * kRows - 1) / (kWaves * kRows);
  hipLaunchKernelGGL(mx4_gather_kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)),
                     dim3(64 * kWaves), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
