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
//   before it in the rows of the step. With a count of pages that steps before have
//   taken, the list starts behind them and the step's are counted on top: a step's
//   count is the next one's, so that steps need no host between them.
// window: query j of a request of L tokens sits at p = L - q_len + j and sees
//   tokens 0 .. f - 1, f = min(first, p + 1), and max(f, p + 1 - window) .. p.
//
// A slot is page * 64 + r % 64; -1 stands where the table (or the free list)
// maps no page. Sums saturate at the largest int32.
#include <algorithm>

#include "remnant_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = RM_MAX_SLOT_BATCH;
constexpr int64_t kMaxPage = (int64_t)1 << 25;  // slots fit in int32
constexpr uint32_t kSat = 0x7fffffff;

struct AppendArgs {
  int32_t* table;
  int64_t table_stride, width;
  const int32_t* old_len;
  const int32_t* new_len;
  int64_t batch;
  uint32_t ratio_m;
  int ratio_shift;
  const int32_t* free_pages;
  int64_t n_free;
  int64_t rows;
  int32_t* loc;
  int32_t* positions;
  int32_t* row_starts;
  int32_t* seqlens;
  int32_t* pages_taken;
  const int32_t* taken;  // of kAfter: pages that the steps before took
};

// Tokens to records, a negative length as 0: floor(x / ratio) for x < 2^31 by a
// product. With 2^s >= ratio and m = ceil(2^(31+s) / ratio) = (2^(31+s) + d) / ratio,
// 0 <= d < ratio, the quotient x m / 2^(31+s) is x / ratio plus x d / (ratio 2^(31+s)),
// less than 1 / ratio since x < 2^31 and d < 2^s; x / ratio lies at least that far
// below the next integer.
__device__ __forceinline__ uint32_t records_of(const AppendArgs& a, int32_t tokens) {
  return (uint32_t)(((uint64_t)(uint32_t)max(tokens, 0) * a.ratio_m) >> a.ratio_shift);
}
__device__ __forceinline__ uint32_t pages_of(uint32_t records) {
  return records / kPageRecords + (records % kPageRecords != 0);
}
__device__ __forceinline__ int32_t slot_in(int64_t page, uint32_t record) {
  return page >= 0 && page < kMaxPage ? (int32_t)(page * kPageRecords + record % kPageRecords) : -1;
}
// Sums saturate at 2^32 - 1 on the way, which the last minimum cannot tell from 2^31 - 1.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return __builtin_elementwise_add_sat(a, b);
}
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t scan_step(uint32_t x) {
  return add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xf, false));
}
// Sum of the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x = scan_step<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8
  x = scan_step<0x112, 0xf>(x);
  x = scan_step<0x114, 0xf>(x);
  x = scan_step<0x118, 0xf>(x);
  x = scan_step<0x142, 0xa>(x);  // row_bcast:15, 31
  return scan_step<0x143, 0xc>(x);
}
// First request whose sum passes i; there is one.
__device__ __forceinline__ int request_of(const int32_t* end, int batch, int32_t i) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (end[mid] > i)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// Every workgroup sums all requests by itself (a few KB of lengths out of L2, the
// sums of its threads scanned by DPP and kept in LDS with the requests' old records)
// and then takes its share of the pages taken and of the rows, each finding its
// request by a binary search in LDS; pages from the last workgroup on, so that a step
// of few rows has them done beside its rows (256 requests, 1 row each: 4.0 -> 3.5 us).
//
// Bound by its chain (lengths, sums, the page's look-up, the row) on a step: 3.4 us in
// a graph whose empty kernels take 2.4; by that and the 8 MB written for 1,048,576
// rows of 16 requests: 5.4 us. With four rows a thread written as one piece these took 5.5
// and 4,096 to 262,144 rows 1.0 us more; with table columns by a wave a request 12.4.
// 1,024 threads a workgroup sum more than kNarrowBatch requests in less time (8,192
// requests 17.9 -> 9.1 us, 1,024 5.1 -> 4.6, 512 4.1 -> 4.0; 256 threads are quicker
// below: 16 requests 3.3 and 3.5). kAfter: behind the pages that steps before took (one
// kernel for both took 0.05 us more of a step's 3.4).
constexpr int64_t kNarrowBatch = 256;
template <int kSize, bool kAfter>
__global__ __launch_bounds__(kSize) void append_slots_kernel(AppendArgs a) {
  extern __shared__ int32_t sm[];
  const int batch = (int)a.batch;
  int32_t* const row_end = sm;              // [batch] rows up to and with request b
  int32_t* const page_end = sm + batch;     // [batch] the same of the pages taken
  int32_t* const held = sm + 2 * batch;     // [batch] records before the step
  __shared__ uint32_t wave_sum[2][kSize / 64];
  const int tid = threadIdx.x, lane = wave_lane(), wave = uniform(tid >> 6);
  const uint32_t gone = kAfter ? (uint32_t)max(*a.taken, 0) : 0;
  // each wave sums its share of the requests, 64 at a time
  const int span = ((batch + kSize - 1) / kSize) * 64;
  const int b0 = min(wave * span, batch), b1 = min(b0 + span, batch);
  uint32_t rows = 0, pages = 0;  // of the wave's requests so far
  for (int t = b0; t < b1; t += 64) {
    const int b = t + lane;
    uint32_t o = 0, n = 0;
    if (b < b1) {
      o = records_of(a, a.old_len[b]);
      n = max(records_of(a, a.new_len[b]), o);
    }
    const uint32_t r = add_sat(wave_scan(n - o), rows);
    const uint32_t p = add_sat(wave_scan(pages_of(n) - pages_of(o)), pages);
    rows = __builtin_amdgcn_readlane(r, 63);
    pages = __builtin_amdgcn_readlane(p, 63);
    if (b < b1) {
      row_end[b] = (int32_t)r;
      page_end[b] = (int32_t)p;
      held[b] = (int32_t)o;
      if (blockIdx.x == 0) a.seqlens[b] = (int32_t)n;
    }
  }
  if (lane == 0) {
    wave_sum[0][wave] = rows;
    wave_sum[1][wave] = pages;
  }
  __syncthreads();
  uint32_t rows_before = 0, pages_before = 0, all_pages = 0;  // of the waves before
  for (int w = 0; w < kSize / 64; ++w) {
    if (w < wave) {
      rows_before = add_sat(rows_before, wave_sum[0][w]);
      pages_before = add_sat(pages_before, wave_sum[1][w]);
    }
    all_pages = add_sat(all_pages, wave_sum[1][w]);
  }
  for (int b = b0 + lane; b < b1; b += 64) {
    const uint32_t r = min(add_sat(rows_before, (uint32_t)row_end[b]), kSat);
    row_end[b] = (int32_t)r;
    page_end[b] = (int32_t)min(add_sat(pages_before, (uint32_t)page_end[b]), kSat);
    if (blockIdx.x == 0) a.row_starts[b + 1] = (int32_t)r;
  }
  all_pages = min(all_pages, kSat);
  if (blockIdx.x == 0 && tid == 0) {
    a.row_starts[0] = 0;
    *a.pages_taken = (int32_t)(kAfter ? min(add_sat(gone, all_pages), kSat) : all_pages);
  }
  const int64_t skip = kAfter ? min((int64_t)gone, a.n_free) : 0;
  const int32_t* const free_pages = a.free_pages + skip;
  const int64_t n_free = a.n_free - skip;
  __syncthreads();
  // the rows
  const int64_t step = (int64_t)gridDim.x * kSize;
  const int64_t total = batch > 0 ? row_end[batch - 1] : 0;
  for (int64_t i = (int64_t)blockIdx.x * kSize + tid; i < a.rows; i += step) {
    const int32_t* from = nullptr;  // where the row's page stands
    uint32_t record = 0;
    if (i < total) {
      const int b = request_of(row_end, batch, (int32_t)i);
      record = (uint32_t)held[b] + (uint32_t)(i - (b > 0 ? row_end[b - 1] : 0));
      const int64_t column = record / kPageRecords, own = pages_of(held[b]);
      const int64_t at = (b > 0 ? page_end[b - 1] : 0) + column - own;
      if (column < a.width) {
        if (column < own)
          from = a.table + b * a.table_stride + column;
        else if (at < n_free)
          from = free_pages + at;
      }
    }
    a.loc[i] = from ? slot_in(*from, record) : -1;
    a.positions[i] = (int32_t)record;
  }
  // the pages, from the last workgroup on: each to its request's next column
  const int64_t first = (int64_t)(gridDim.x - 1 - blockIdx.x) * kSize + tid;
  for (int64_t i = first; i < min((int64_t)all_pages, n_free); i += step) {
    const int b = request_of(page_end, batch, (int32_t)i);
    const int64_t c = (int64_t)pages_of(held[b]) + i - (b > 0 ? page_end[b - 1] : 0);
    if (c < a.width) a.table[b * a.table_stride + c] = free_pages[i];
  }
  if (all_pages > n_free) {  // too few: -1 in the columns left over, a wave a request
    for (int64_t b = first / 64; b < batch; b += step / 64) {
      const uint32_t o = held[b];
      const int64_t base = b > 0 ? page_end[b - 1] : 0;
      const uint32_t n = max(records_of(a, a.new_len[b]), o);
      const int64_t from = pages_of(o), to = min((int64_t)pages_of(n), a.width);
      for (int64_t c = from + max(n_free - base, (int64_t)0) + lane; c < to; c += 64)
        a.table[b * a.table_stride + c] = -1;
    }
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

// A thread takes kVec entries of one token and asks for their pages at once. Bound by
// the chain length, page, entry on a step (256 requests x 2 tokens x 132 entries 2.8 us,
// 2.4 an empty kernel), by the written bytes on long lists (8 x 131,072 entries, 4 MB,
// 4.0 us; 64 x 131,072, 34 MB, 15). Four entries a thread from kFourEntries on where
// rows divide: 131,072 entries 2.8 us with one and 3.2 with four, 262,144 3.4 and 3.2,
// 1,048,576 6.2 and 4.2.
constexpr int64_t kFourEntries = 1 << 18;
template <int kVec>
__global__ __launch_bounds__(kThreads) void window_slots_kernel(WindowArgs a) {
  const int64_t out_width = a.first + a.window;
  const int64_t across = max((out_width + kVec - 1) / kVec, (int64_t)1);  // threads a token
  const int64_t all = a.batch * a.q_len * across;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < all;
       e += (int64_t)gridDim.x * kThreads) {
    int64_t t, b;
    if (all <= 0xffffffffll) {
      t = (uint32_t)e / (uint32_t)across;
      b = (uint32_t)t / (uint32_t)a.q_len;
    } else {
      t = e / across;
      b = t / a.q_len;
    }
    const int64_t i0 = (e - t * across) * kVec;
    const int64_t p = (int64_t)a.lengths[b] - a.q_len + (t - b * a.q_len);
    const int64_t f = max(min(a.first, p + 1), (int64_t)0);
    const int64_t start = max(f, p + 1 - a.window);
    const int64_t count = p < 0 ? 0 : f + p + 1 - start;
    if (i0 == 0) a.counts[t] = (int32_t)count;
    typedef int32_t Vec __attribute__((ext_vector_type(kVec)));
    Vec slot;
    const int32_t* const row = a.table + b * a.table_stride;
    uint32_t token[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const int64_t i = i0 + v;
      token[v] = (uint32_t)(i < f ? i : start + i - f);
      slot[v] = -1;
      if (i < count && token[v] / kPageRecords < a.width) slot[v] = row[token[v] / kPageRecords];
    }
#pragma unroll
    for (int v = 0; v < kVec; ++v) slot[v] = slot_in(slot[v], token[v]);
    if (i0 < out_width) *(Vec*)(a.slots + t * out_width + i0) = slot;
  }
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

// Whether [p, p + n) and [q, q + m) int32 elements share memory.
bool overlap(const int32_t* p, int64_t n, const int32_t* q, int64_t m) {
  return n > 0 && m > 0 && (uintptr_t)p < (uintptr_t)(q + m) && (uintptr_t)q < (uintptr_t)(p + n);
}

}  // namespace

extern "C" int rm_append_slots_after(int32_t* block_table, int64_t block_table_stride,
                                     int64_t max_blocks, const int32_t* old_lengths,
                                     const int32_t* new_lengths, int64_t batch, int64_t ratio,
                                     const int32_t* free_pages, int64_t n_free,
                                     const int32_t* taken, int64_t rows, int32_t* loc,
                                     int32_t* positions, int32_t* row_starts, int32_t* seqlens,
                                     int32_t* pages_taken, void* stream) {
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
                        (const void*)row_starts, (const void*)seqlens, (const void*)pages_taken,
                        (const void*)taken})
    if (!aligned(p, 4)) return RM_ERR_ALIGN;
  // what is written must be apart from what other workgroups still read, and from each other
  const int64_t table_n = batch > 0 ? (batch - 1) * block_table_stride + max_blocks : 0;
  const struct {
    const int32_t* p;
    int64_t n;
  } in[4] = {{old_lengths, batch}, {new_lengths, batch}, {free_pages, n_free}, {taken, taken ? 1 : 0}},
    out[6] = {{block_table, table_n}, {loc, rows},       {positions, rows},
              {row_starts, batch + 1}, {seqlens, batch}, {pages_taken, 1}};
  for (int i = 0; i < 6; ++i) {
    for (int j = 0; j < 4; ++j)
      if (overlap(out[i].p, out[i].n, in[j].p, in[j].n)) return RM_ERR_SHAPE;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return RM_ERR_SHAPE;
  }
  int log2 = 0;  // 2^log2 >= ratio
  while (((int64_t)1 << log2) < ratio) ++log2;
  const uint32_t m = (uint32_t)((((uint64_t)1 << (31 + log2)) + ratio - 1) / ratio);
  AppendArgs a{block_table, block_table_stride, max_blocks, old_lengths, new_lengths, batch, m,
               31 + log2, free_pages, n_free, rows, loc, positions, row_starts, seqlens,
               pages_taken, taken};
  const bool wide = batch > kNarrowBatch;
  const int64_t threads = wide ? 1024 : kThreads;
  const int64_t lds = batch * 3 * sizeof(int32_t);
  // as many as run at once
  const int64_t most = 256 * std::min<int64_t>(2048 / threads / 2, 160 * 1024 / (lds + 1024));
  const int64_t blocks = std::min<int64_t>((rows + threads - 1) / threads + 1, most);
  const auto kern =
      wide ? (taken ? append_slots_kernel<1024, true> : append_slots_kernel<1024, false>)
           : (taken ? append_slots_kernel<kThreads, true> : append_slots_kernel<kThreads, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3((unsigned)threads), (size_t)lds,
                     (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}

extern "C" int rm_append_slots(int32_t* block_table, int64_t block_table_stride,
                               int64_t max_blocks, const int32_t* old_lengths,
                               const int32_t* new_lengths, int64_t batch, int64_t ratio,
                               const int32_t* free_pages, int64_t n_free, int64_t rows,
                               int32_t* loc, int32_t* positions, int32_t* row_starts,
                               int32_t* seqlens, int32_t* pages_taken, void* stream) {
  return rm_append_slots_after(block_table, block_table_stride, max_blocks, old_lengths,
                               new_lengths, batch, ratio, free_pages, n_free, nullptr, rows, loc,
                               positions, row_starts, seqlens, pages_taken, stream);
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
  const int64_t row = first + window;
  const bool four = row % 4 == 0 && aligned(slots, 16) && tokens * row >= kFourEntries;
  const int64_t across = std::max<int64_t>(row / (four ? 4 : 1), 1);
  const int64_t blocks = (tokens * across + kThreads - 1) / kThreads;
  hipLaunchKernelGGL((four ? window_slots_kernel<4> : window_slots_kernel<1>),
                     dim3((unsigned)std::min<int64_t>(blocks, 16384)), dim3(kThreads), 0,
                     (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
