// Block tables and slot maps, built on the GPU from the requests' lengths: the
// int32 inputs that the store (slots, positions), the readers (slot lists) and
// the decode (block table, record counts, window slots) of this library take.
//
// append: request b holds o = old / ratio records before the step and
//   n = max(new / ratio, o) after it (lengths in tokens, negative ones 0).
//   With P(r) = ceil(r / 64) pages for r records it takes P(n) - P(o) pages,
//   the requests in order, from the front of the free list: column c of row b,
//   P(o) <= c < P(n), becomes free[base_b + c - P(o)], base_b the exclusive sum
//   of the pages taken. Its new records o .. n - 1 follow those of the requests
//   before it in the rows of the step.
// window: query j of a request of L tokens sits at p = L - q_len + j and sees
//   tokens 0 .. f - 1, f = min(first, p + 1), and max(f, p + 1 - window) .. p.
//
// A slot is page * 64 + r % 64; -1 stands where the table (or the free list)
// maps no page. All sums are 64-bit and saturate at the largest int32.
#include <algorithm>

#include "remnant_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = RM_MAX_SLOT_BATCH;
constexpr int64_t kMaxPage = (int64_t)1 << 25;  // slots fit in int32
constexpr int64_t kSat = 0x7fffffff;

struct AppendArgs {
  int32_t* table;
  int64_t table_stride, width;
  const int32_t* old_len;
  const int32_t* new_len;
  int64_t batch;
  uint32_t ratio;
  const int32_t* free_pages;
  int64_t n_free;
  int64_t rows;
  int32_t* loc;
  int32_t* positions;
  int32_t* row_starts;
  int32_t* seqlens;
  int32_t* pages_taken;
};

__device__ __forceinline__ int64_t pages_of(int64_t records) {
  return (records + kPageRecords - 1) / kPageRecords;
}
__device__ __forceinline__ int32_t slot_in(int64_t page, int64_t record) {
  return page >= 0 && page < kMaxPage ? (int32_t)(page * kPageRecords + record % kPageRecords) : -1;
}
__device__ __forceinline__ void records_of(const AppendArgs& a, int64_t b, int64_t& o, int64_t& n) {
  o = (uint32_t)max(a.old_len[b], 0) / a.ratio;
  n = max((int64_t)((uint32_t)max(a.new_len[b], 0) / a.ratio), o);
}

// Every workgroup sums all requests by itself (a few KB of lengths out of L2)
// and then takes its share of the rows; requests' table columns go by waves.
__global__ __launch_bounds__(kThreads) void append_slots_kernel(AppendArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* const row_end = sm;             // [batch] rows up to and with request b
  int32_t* const page_end = sm + a.batch;  // [batch] the same of the pages taken
  __shared__ int64_t part[2][kThreads];
  const int tid = threadIdx.x;
  const int64_t per = (a.batch + kThreads - 1) / kThreads;
  const int64_t b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t rows = 0, pages = 0;
  for (int64_t b = b0; b < b1; ++b) {
    int64_t o, n;
    records_of(a, b, o, n);
    rows += n - o;
    pages += pages_of(n) - pages_of(o);
    row_end[b] = (int32_t)min(rows, kSat);
    page_end[b] = (int32_t)min(pages, kSat);
  }
  part[0][tid] = rows;
  part[1][tid] = pages;
  __syncthreads();
  for (int d = 1; d < kThreads; d *= 2) {
    const int64_t r = tid >= d ? part[0][tid - d] : 0, p = tid >= d ? part[1][tid - d] : 0;
    __syncthreads();
    part[0][tid] += r;
    part[1][tid] += p;
    __syncthreads();
  }
  const int64_t rows_before = part[0][tid] - rows, pages_before = part[1][tid] - pages;
  for (int64_t b = b0; b < b1; ++b) {
    row_end[b] = (int32_t)min(rows_before + row_end[b], kSat);
    page_end[b] = (int32_t)min(pages_before + page_end[b], kSat);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int64_t b = tid; b < a.batch; b += kThreads) {
      int64_t o, n;
      records_of(a, b, o, n);
      a.seqlens[b] = (int32_t)n;
      a.row_starts[b + 1] = row_end[b];
    }
    if (tid == 0) {
      a.row_starts[0] = 0;
      *a.pages_taken = a.batch > 0 ? page_end[a.batch - 1] : 0;
    }
  }
  // the new columns: a wave a request
  const int lane = wave_lane();
  const int64_t waves = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 64) + tid / 64; b < a.batch; b += waves) {
    int64_t o, n;
    records_of(a, b, o, n);
    const int64_t base = b > 0 ? page_end[b - 1] : 0, held = pages_of(o);
    const int64_t end = min(pages_of(n), a.width);
    for (int64_t c = held + lane; c < end; c += 64) {
      const int64_t at = base + c - held;
      a.table[b * a.table_stride + c] = at < a.n_free ? a.free_pages[at] : -1;
    }
  }
  // the rows: their request by binary search
  const int64_t total = a.batch > 0 ? row_end[a.batch - 1] : 0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < a.rows;
       i += (int64_t)gridDim.x * kThreads) {
    int32_t slot = -1, position = 0;
    if (i < total) {
      int64_t lo = 0, hi = a.batch - 1;  // first request whose rows end behind i
      while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (row_end[mid] > i)
          hi = mid;
        else
          lo = mid + 1;
      }
      int64_t o, n;
      records_of(a, lo, o, n);
      const int64_t record = o + i - (lo > 0 ? row_end[lo - 1] : 0);
      const int64_t column = record / kPageRecords, held = pages_of(o);
      int64_t page = -1;
      if (column < a.width) {
        if (column < held) {
          page = a.table[lo * a.table_stride + column];
        } else {
          const int64_t at = (lo > 0 ? page_end[lo - 1] : 0) + column - held;
          page = at < a.n_free ? a.free_pages[at] : -1;
        }
      }
      slot = slot_in(page, record);
      position = (int32_t)record;
    }
    a.loc[i] = slot;
    a.positions[i] = position;
  }
}

struct WindowArgs {
  const int32_t* table;
  int64_t table_stride, width;
  const int32_t* lengths;
  int64_t batch, q_len, window, first;
  int32_t* slots;
  int32_t* counts;
};

__global__ __launch_bounds__(kThreads) void window_slots_kernel(WindowArgs a) {
  const int64_t tokens = a.batch * a.q_len, out_width = a.first + a.window;
  for (int64_t t = blockIdx.y; t < tokens; t += gridDim.y) {
    const int64_t b = t / a.q_len;
    const int64_t p = (int64_t)a.lengths[b] - a.q_len + (t - b * a.q_len);
    const int64_t f = max(min(a.first, p + 1), (int64_t)0);
    const int64_t start = max(f, p + 1 - a.window);
    const int64_t count = p < 0 ? 0 : f + p + 1 - start;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.counts[t] = (int32_t)count;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < out_width;
         i += (int64_t)gridDim.x * kThreads) {
      int32_t slot = -1;
      if (i < count) {
        const int64_t token = i < f ? i : start + i - f;
        const int64_t column = token / kPageRecords;
        if (column < a.width) slot = slot_in(a.table[b * a.table_stride + column], token);
      }
      a.slots[t * out_width + i] = slot;
    }
  }
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

// Whether [p, p + n) and [q, q + m) int32 elements share memory.
bool overlap(const int32_t* p, int64_t n, const int32_t* q, int64_t m) {
  return n > 0 && m > 0 && (uintptr_t)p < (uintptr_t)(q + m) && (uintptr_t)q < (uintptr_t)(p + n);
}

}  // namespace

extern "C" int rm_append_slots(int32_t* block_table, int64_t block_table_stride,
                               int64_t max_blocks, const int32_t* old_lengths,
                               const int32_t* new_lengths, int64_t batch, int64_t ratio,
                               const int32_t* free_pages, int64_t n_free, int64_t rows,
                               int32_t* loc, int32_t* positions, int32_t* row_starts,
                               int32_t* seqlens, int32_t* pages_taken, void* stream) {
  if (batch < 0 || batch > kMaxBatch || max_blocks < 0 || n_free < 0 || rows < 0 || rows > kSat ||
      max_blocks > kSat || n_free > kSat || ratio < 1 || ratio > kSat ||
      (batch > 1 && block_table_stride < max_blocks))
    return RM_ERR_SHAPE;
  if (!row_starts || !pages_taken || (batch > 0 && (!old_lengths || !new_lengths || !seqlens)) ||
      (batch > 0 && max_blocks > 0 && !block_table) || (n_free > 0 && !free_pages) ||
      (rows > 0 && (!loc || !positions)))
    return RM_ERR_NULL;
  for (const void* p : {(const void*)block_table, (const void*)old_lengths, (const void*)new_lengths,
                        (const void*)free_pages, (const void*)loc, (const void*)positions,
                        (const void*)row_starts, (const void*)seqlens, (const void*)pages_taken})
    if (!aligned(p, 4)) return RM_ERR_ALIGN;
  // what is written must be apart from what other workgroups still read, and from each other
  const int64_t table_n = batch > 0 ? (batch - 1) * block_table_stride + max_blocks : 0;
  const struct {
    const int32_t* p;
    int64_t n;
  } in[3] = {{old_lengths, batch}, {new_lengths, batch}, {free_pages, n_free}},
    out[6] = {{block_table, table_n}, {loc, rows},       {positions, rows},
              {row_starts, batch + 1}, {seqlens, batch}, {pages_taken, 1}};
  for (int i = 0; i < 6; ++i) {
    for (int j = 0; j < 3; ++j)
      if (overlap(out[i].p, out[i].n, in[j].p, in[j].n)) return RM_ERR_SHAPE;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return RM_ERR_SHAPE;
  }
  AppendArgs a{block_table, block_table_stride, max_blocks, old_lengths, new_lengths, batch,
               (uint32_t)ratio, free_pages, n_free, rows, loc, positions, row_starts, seqlens,
               pages_taken};
  int64_t blocks = std::max((rows + 4 * kThreads - 1) / (4 * kThreads), (batch + 31) / 32);
  blocks = std::min<int64_t>(std::max<int64_t>(blocks, 1), 256);
  hipLaunchKernelGGL(append_slots_kernel, dim3((unsigned)blocks), dim3(kThreads),
                     (size_t)batch * 2 * sizeof(int32_t), (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}

extern "C" int rm_window_slots(const int32_t* block_table, int64_t block_table_stride,
                               int64_t max_blocks, const int32_t* lengths, int64_t batch,
                               int64_t q_len, int64_t window, int64_t first, int32_t* slots,
                               int32_t* counts, void* stream) {
  if (batch < 0 || q_len < 0 || window < 0 || first < 0 || max_blocks < 0 || window > kSat ||
      first > kSat || q_len > kSat || batch > kSat || max_blocks > kSat || first + window > kSat ||
      (batch > 1 && block_table_stride < max_blocks))
    return RM_ERR_SHAPE;
  const int64_t tokens = batch * q_len;
  if (tokens > kSat) return RM_ERR_SHAPE;
  if (tokens == 0) return RM_OK;
  if (!lengths || !counts || (first + window > 0 && !slots) || (max_blocks > 0 && !block_table))
    return RM_ERR_NULL;
  for (const void* p : {(const void*)block_table, (const void*)lengths, (const void*)slots,
                        (const void*)counts})
    if (!aligned(p, 4)) return RM_ERR_ALIGN;
  const int64_t table_n = (batch - 1) * block_table_stride + max_blocks;
  const int64_t n = tokens * (first + window);
  if (overlap(slots, n, block_table, table_n) || overlap(slots, n, lengths, batch) ||
      overlap(counts, tokens, block_table, table_n) || overlap(counts, tokens, lengths, batch) ||
      overlap(slots, n, counts, tokens))
    return RM_ERR_SHAPE;
  WindowArgs a{block_table, block_table_stride, max_blocks, lengths, batch, q_len, window, first,
               slots, counts};
  const int64_t across = std::max<int64_t>((first + window + kThreads - 1) / kThreads, 1);
  const dim3 grid((unsigned)std::min<int64_t>(across, 1024), (unsigned)std::min<int64_t>(tokens, 65535));
  hipLaunchKernelGGL(window_slots_kernel, grid, dim3(kThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
