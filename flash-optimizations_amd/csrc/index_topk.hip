// Selection of the k highest of each row's first length scores, as ascending record
// numbers: equal scores go to the lowest records, NaN counts as -inf.
//
// A workgroup takes a row. Scores become keys whose unsigned order is theirs. The k-th
// highest key lies in [lo, hi], at first the row's smallest and largest; a histogram of
// that range in 2,048 equal bins (in LDS) finds its bin, which is the next range, until
// the bin is taken whole or is one key: at most three histograms, as each leaves 11 bits
// fewer. Range by range and not by fixed digits, since scores of one query share most of
// their leading bits. Then every wave counts what it takes of each turn of 256 scores,
// a scan over turns and waves gives the places, and the numbers are written in order.
#include <algorithm>

#include "remnant_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kBins = 2048;
constexpr uint32_t kLowestKey = 0x007fffffu;  // of -inf, and of NaN; 0 is no score

struct TopkArgs {
  const float* scores;
  int64_t stride;
  const int32_t* lengths;  // null: width
  int width, k;
  bool wide;  // rows are 16-byte aligned
  int32_t *indices, *counts;
};

__device__ __forceinline__ uint32_t key_of(float x) {
  const int b = (int)f2u(x + 0.0f);  // (-0 and 0 are equal)
  const uint32_t key = (uint32_t)(b ^ ((b >> 31) | (int)0x80000000u));
  return x != x ? kLowestKey : key;
}

template <int kThreads>
struct Shared {
  static constexpr int kWaves = kThreads / 64;
  uint32_t bins[kBins];
  uint32_t part[2 * kWaves];
  uint32_t pick[4];
};

__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x = min(x, (uint32_t)__shfl_xor((int)x, d, 64));
  return x;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, d, 64));
  return x;
}
// Inclusive sum over the wave's lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x) {
  const int lane = wave_lane();
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t y = (uint32_t)__shfl_up((int)x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}
__device__ __forceinline__ int below(uint64_t mask) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// kHeld: turns of 4 * kThreads scores that the row's keys stay in registers for; 0: a row of
// any length, read again for each pass.
template <int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads) void index_topk_kernel(TopkArgs a) {
  using S = Shared<kThreads>;
  __shared__ S s;
  const int tid = (int)threadIdx.x, lane = wave_lane(), wave = uniform(tid >> 6);
  const int64_t row = blockIdx.x;
  const int length = a.lengths ? min(max(a.lengths[row], 0), a.width) : a.width;
  const int count = min(length, a.k);
  int32_t* const out = a.indices + row * a.k;
  if (tid == 0) a.counts[row] = count;
  for (int i = count + tid; i < a.k; i += kThreads) out[i] = -1;
  if (count == length) {
    for (int i = tid; i < count; i += kThreads) out[i] = i;
    return;
  }
  if (count == 0) return;
  const float* const from = a.scores + row * a.stride;
  const int turns = (length + 4 * kThreads - 1) / (4 * kThreads);
  auto load = [&](int turn, uint32_t (&key)[4]) {
    const int at = 4 * (turn * kThreads + tid);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.wide && at + 3 < length) {
      const f32x4 v = *(const f32x4*)(from + at);
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = v[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (at + c < length) x[c] = from[at + c];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) key[c] = at + c < length ? key_of(x[c]) : 0u;
  };
  uint32_t held[kHeld > 0 ? kHeld : 1][4];
  // f(turn, keys) for every turn of the row
  auto each = [&](auto f) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (i < turns) f(i, held[i]);
    } else {
      for (int i = 0; i < turns; ++i) {
        uint32_t key[4];
        load(i, key);
        f(i, key);
      }
    }
  };
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i < turns) load(i, held[i]);
  }
  // the range of all keys
  uint32_t lo = 0xffffffffu, hi = 0;
  each([&](int, const uint32_t (&key)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      hi = max(hi, key[c]);
      lo = min(lo, key[c] != 0 ? key[c] : 0xffffffffu);
    }
  });
  lo = wave_min(lo);
  hi = wave_max(hi);
  if (lane == 0) s.part[wave] = lo, s.part[S::kWaves + wave] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < S::kWaves; ++w) {
    lo = min(lo, s.part[w]);
    hi = max(hi, s.part[S::kWaves + w]);
  }
  // need: how many of [lo, hi] are taken; those above hi are taken whole
  uint32_t need = (uint32_t)count;
  for (;;) {
    if (lo == hi) break;
    const int bits = 32 - __builtin_clz(hi - lo);
    const int shift = max(bits - 11, 0);
    for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
    __syncthreads();
    each([&](int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (key[c] >= lo && key[c] <= hi) atomicAdd(&s.bins[(key[c] - lo) >> shift], 1u);
    });
    __syncthreads();
    // the bin that holds the need-th from above: thread t sums bins from the top
    constexpr int kPer = kBins / kThreads;
    uint32_t mine[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      mine[i] = s.bins[kBins - 1 - (tid * kPer + i)];
      sum += mine[i];
    }
    const uint32_t upto = wave_prefix(sum);
    if (lane == 63) s.part[wave] = upto;
    __syncthreads();
    uint32_t before = upto - sum;
    for (int w = 0; w < wave; ++w) before += s.part[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (before < need && before + mine[i] >= need) {
        s.pick[0] = (uint32_t)(kBins - 1 - (tid * kPer + i));
        s.pick[1] = before;
        s.pick[2] = mine[i];
      }
      before += mine[i];
    }
    __syncthreads();
    const uint32_t bin = s.pick[0], held_in = s.pick[2];
    need -= s.pick[1];
    lo += bin << shift;
    hi = min(hi, lo + ((1u << shift) - 1));
    if (held_in == need) break;  // the bin is taken whole
    __syncthreads();             // (bins and pick are written again)
  }
  // Taken: keys above hi, and of [lo, hi] the first `need`. (A range that is taken whole
  // has just as many; else it is one key.)
  __syncthreads();
  uint32_t above = 0, ties = 0;  // of the turns before
  each([&](int turn, const uint32_t (&key)[4]) {
    uint64_t over[4], same[4];
    uint32_t n_over = 0, n_same = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      over[c] = __ballot(key[c] > hi);
      same[c] = __ballot(key[c] >= lo && key[c] <= hi);
      n_over += __popcll(over[c]);
      n_same += __popcll(same[c]);
    }
    uint32_t* const part = s.bins + (turn & 1) * 2 * S::kWaves;
    if (lane == 0) part[2 * wave] = n_over, part[2 * wave + 1] = n_same;
    __syncthreads();
    uint32_t a0 = above, t0 = ties;
#pragma unroll
    for (int w = 0; w < S::kWaves; ++w) {
      const uint32_t o = part[2 * w], e = part[2 * w + 1];
      if (w < wave) a0 += o, t0 += e;
      above += o;
      ties += e;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      a0 += below(over[c]);
      t0 += below(same[c]);
    }
    const int at = 4 * (turn * kThreads + tid);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool is_over = key[c] > hi, is_same = key[c] >= lo && key[c] <= hi;
      if (is_over || (is_same && t0 < need)) out[a0 + min(t0, need)] = at + c;
      a0 += is_over;
      t0 += is_same;
    }
  });
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

}  // namespace

extern "C" int rm_index_topk(const float* scores, int64_t row_stride, const int32_t* lengths,
                             int64_t rows, int64_t width, int64_t k, int32_t* indices,
                             int32_t* counts, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || width < 0 || width > RM_MAX_INDEX_WIDTH || k < 0 ||
      k > RM_MAX_INDEX_WIDTH || (rows > 1 && row_stride < width))
    return RM_ERR_SHAPE;
  if (rows == 0) return RM_OK;
  if (!counts || (width > 0 && !scores) || (k > 0 && !indices)) return RM_ERR_NULL;
  if (!aligned(scores, 4) || !aligned(lengths, 4) || !aligned(indices, 4) || !aligned(counts, 4))
    return RM_ERR_ALIGN;
  const TopkArgs a{scores, row_stride, lengths, (int)width, (int)k,
                   aligned(scores, 16) && (rows == 1 || row_stride % 4 == 0), indices, counts};
  const auto kern = width <= 2048    ? index_topk_kernel<256, 2>
                    : width <= 8192  ? index_topk_kernel<1024, 2>
                    : width <= 32768 ? index_topk_kernel<1024, 8>
                                     : index_topk_kernel<1024, 0>;
  hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3(width <= 2048 ? 256 : 1024), 0,
                     (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? RM_OK : RM_ERR_LAUNCH;
}
