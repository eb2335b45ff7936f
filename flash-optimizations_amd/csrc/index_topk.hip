// Selection of the k highest of each row's first length scores, as ascending record
// numbers: equal scores go to the lowest records, NaN counts as -inf.
//
// A workgroup takes a row. Scores become keys whose unsigned order is theirs, held in
// registers (and LDS, for long rows): the row is read once. The k-th highest key lies in
// [lo, hi]: from the lowest of the threads' highest or second highest keys, which enough
// keys reach (it leaves a quarter of a row of ordinary scores), to the highest. A histogram of
// that range in 2,048 equal bins (in LDS) finds its bin; a bin of up to 64 keys is listed
// and ranked, a larger one is the next range: at most three histograms, as each leaves 11
// bits fewer. Range by range and not by fixed digits, since scores of one query share most
// of their leading bits. A wave's scores stand together, so that each wave knows its places
// from one count a wave; numbers are put in order in LDS and written side by side.
//
// Bound by one workgroup a CU, whose phases wait for each other: loads, then about thirty vector
// operations a key (seven make it and find the range while the row comes) in passes with a
// barrier between them. Vector instructions are issued in half of the busy cycles (256 rows of
// 32,768: 16.2 us, 512 rows 30.3; 512 of 35,840 39.3; 64 ragged rows of up to 32,768 11.5, on 64
// of 256 CUs; one of 8,192 6.0, a launch and six barriers).
#include <algorithm>

#include "remnant_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kBins = 2048;
// (Keys are 0x007fffff, of -inf, and up: 0 is no score.)

struct TopkArgs {
  const float* scores;
  int64_t stride;
  const int32_t* lengths;  // null: width
  int width, k;
  bool wide;  // rows are 16-byte aligned
  int32_t *indices, *counts;
};

__device__ __forceinline__ uint32_t key_of(float x) {
  // (the sum makes -0 zero and any NaN quiet, the maximum NaN -inf)
  const int b = (int)f2u(fmaxf(x + 0.0f, -INFINITY));
  return (uint32_t)(b ^ ((b >> 31) | (int)0x80000000u));
}
__device__ __forceinline__ uint32_t least(uint32_t x, uint32_t y) { return min(x, y); }
__device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) { return max(x, y); }
__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return x + y; }

template <int kThreads>
struct Shared {
  static constexpr int kWaves = kThreads / 64;
  uint32_t bins[kBins];  // later the numbers, where they fit
  alignas(16) uint32_t part[5][kWaves];
  uint32_t pick[4];
  u32x2 list[64];        // key, wave
  uint32_t rank[2][64];  // list keys above it, and equal
};

// Over each row of 16 lanes, and over the wave's lanes.
template <class F>
__device__ __forceinline__ uint32_t row_all_of(uint32_t x, F op) {
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, false));
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, false));
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, false));
  return op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, false));
}
template <class F>
__device__ __forceinline__ uint32_t wave_all_of(uint32_t x, F op) {
  x = row_all_of(x, op);
  const auto h = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = op(h[0], h[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return op(q[0], q[1]);
}
// `plus` and how many of the lanes before are in the mask.
__device__ __forceinline__ uint32_t below(uint64_t mask, uint32_t plus) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, plus));
}

// A row's keys stay in registers for kHeld turns of 4 * kThreads scores: as few as hold the
// width, as a turn more is code to fetch and keys to make (1,430 rows of 16,384: 35 us with
// four turns, 65 with eight). kLong: longer rows, with kInLds turns in LDS and what is longer
// still read again for each pass (64 rows of 65,536 23.6 us, 38.4 when each pass read them;
// 256 rows of 32,768 then 6.4 us more when each pass read them).
constexpr int kInLds = 8;
template <int kThreads, int kHeld, bool kLong>
__global__ __launch_bounds__(kThreads) void index_topk_kernel(TopkArgs a) {
  __shared__ u32x4 kept[kLong ? kInLds : 1][kLong ? kThreads : 1];
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
  // a wave's scores stand together, 256 a turn, so that only totals of waves meet; shares
  // differ by less than four scores, so that no thread goes without where others have two turns
  const int share = ((length + 4 * S::kWaves - 1) / (4 * S::kWaves)) * 4;
  const int begin = min(wave * share, length), end = min(begin + share, length);
  const int turns = (share + 255) / 256;
  // A turn's scores as they are, then their keys: in two steps, and with no load left out
  // where there is no score (the row's last whole four instead), so that the keys of one
  // turn need not wait for the loads of another. The row's last scores that are no four
  // (`odd`, from `rest` on) are loaded apart.
  const bool wide = a.wide && length >= 4;
  const int rest = wide ? length & ~3 : 0x7fffffff;
  uint32_t odd[3];
#pragma unroll
  for (int c = 0; c < 3; ++c) odd[c] = f2u(from[min((length & ~3) + c, length - 1)]);
  auto load = [&](int turn, uint32_t (&x)[4]) {
    const int at = begin + 256 * turn + 4 * lane;
    if (wide) {
      const u32x4 v = *(const u32x4*)(from + min(at, (length - 4) & ~3));
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = v[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = f2u(from[min(at + c, length - 1)]);
    }
  };
  auto keys = [&](int turn, uint32_t (&x)[4]) {
    const int at = begin + 256 * turn + 4 * lane;
    const bool last = begin + 256 * (turn + 1) > end;
    if (last && at == rest) {
#pragma unroll
      for (int c = 0; c < 3; ++c) x[c] = odd[c];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = key_of(u2f(x[c]));
    if (last) {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = at + c < end ? x[c] : 0u;
    }
  };
  uint32_t held[kHeld][4];
  // f(turn, keys) for every turn of the row
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i < turns) f(i, held[i]);
    if constexpr (kLong) {
      for (int i = kHeld; i < min(turns, kHeld + kInLds); ++i) {
        const u32x4 x = kept[i - kHeld][tid];
        const uint32_t key[4] = {x[0], x[1], x[2], x[3]};
        f(i, key);
      }
      for (int i = kHeld + kInLds; i < turns; ++i) {
        uint32_t key[4];
        load(i, key);
        keys(i, key);
        f(i, key);
      }
    }
  };
  // The range: from the lowest of the threads' highest keys (the second highest, for more
  // than a key a thread), which enough keys reach, to the highest. Where a thread has none
  // or more are wanted, from the row's lowest key.
  uint32_t lo, hi = 0, second = 0;
  const auto range = [&](int, const uint32_t (&key)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      second = max(second, min(hi, key[c]));  // (hi is not below it: the middle of three)
      hi = max(hi, key[c]);
    }
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) load(i, held[i]);
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    keys(i, held[i]);
    range(i, held[i]);
  }
  if constexpr (kLong) {
    uint32_t key[kInLds][4];
#pragma unroll
    for (int i = 0; i < kInLds; ++i) load(kHeld + i, key[i]);
#pragma unroll
    for (int i = 0; i < kInLds; ++i) {
      keys(kHeld + i, key[i]);
      range(kHeld + i, key[i]);
      kept[i][tid] = u32x4{key[i][0], key[i][1], key[i][2], key[i][3]};
    }
    for (int i = kHeld + kInLds; i < turns; ++i) {
      load(i, key[0]);
      keys(i, key[0]);
      range(i, key[0]);
    }
  }
  lo = wave_all_of(count <= kThreads ? hi : count <= 2 * kThreads ? second : 0u, least);
  hi = wave_all_of(hi, most);
  if (lane == 0) s.part[0][wave] = lo, s.part[1][wave] = hi;
  __syncthreads();
  const int other = lane & (S::kWaves - 1);  // a wave a lane, in each row of 16
  const bool earlier = other < wave && (lane & 15) < S::kWaves;
  static_assert(S::kWaves <= 16, "a row of lanes");
  lo = uniform((int)row_all_of(s.part[0][other], least));
  hi = uniform((int)row_all_of(s.part[1][other], most));
  if (lo == 0) {
    lo = 0xffffffffu;
    each([&](int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) lo = min(lo, key[c] - 1);  // (no score: passed over)
    });
    lo = wave_all_of(lo, least);
    if (lane == 0) s.part[2][wave] = lo;
    __syncthreads();
    lo = uniform((int)row_all_of(s.part[2][other], least)) + 1;
  }
  // need: how many of [lo, hi] are taken; those above hi are taken whole
  uint32_t need = (uint32_t)count;
  bool whole = false;            // all of [lo, hi] are taken
  uint32_t above = 0, ties = 0;  // of the waves before: above hi, and in [lo, hi]
  bool counted = false;
  for (;;) {
    if (lo == hi) break;
    const int bits = 32 - __builtin_clz(hi - lo);
    const int shift = max(bits - 11, 0);
    for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
    if (tid == 0) s.pick[3] = 0;
    if (tid < 128) s.rank[tid >> 6][tid & 63] = 0;
    __syncthreads();
    each([&](int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (key[c] - lo <= hi - lo) atomicAdd(&s.bins[(key[c] - lo) >> shift], 1u);
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
    if (lane == 63) s.part[0][wave] = upto;
    __syncthreads();
    uint32_t before = upto - sum + row_all_of(earlier ? s.part[0][other] : 0u, plus);
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
    if (held_in <= 64) {  // a lane each, ranked by all waves
      uint32_t n_over = 0;
      each([&](int, const uint32_t (&key)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          n_over += __popcll(__ballot(key[c] > hi));
          if (key[c] - lo <= hi - lo)
            s.list[atomicAdd(&s.pick[3], 1u)] = u32x2{key[c], (uint32_t)wave};
        }
      });
      if (lane == 0) s.part[3][wave] = n_over;
      __syncthreads();
      const u32x2 at = lane < (int)held_in ? s.list[lane] : u32x2{0u, 0xffffu};
      uint32_t over = 0, same = 0;
      for (int i = wave; i < (int)held_in; i += S::kWaves) {
        const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)at[0], i);
        over += other > at[0];
        same += other == at[0];
      }
      atomicAdd(&s.rank[0][lane], over);
      atomicAdd(&s.rank[1][lane], same);
      __syncthreads();
      over = s.rank[0][lane], same = s.rank[1][lane];
      // (lanes without a key have all of the others above them)
      const int last = __builtin_ctzll(__ballot(over < need && over + same >= need));
      lo = hi = (uint32_t)__builtin_amdgcn_readlane((int)at[0], last);
      need -= (uint32_t)__builtin_amdgcn_readlane((int)over, last);
      whole = need == (uint32_t)__builtin_amdgcn_readlane((int)same, last);
      above = __popcll(__ballot(at[0] > hi && (int)at[1] < wave));
      ties = __popcll(__ballot(at[0] == hi && (int)at[1] < wave));
      above += row_all_of(earlier ? s.part[3][other] : 0u, plus);
      counted = true;
      break;
    }
    whole = held_in == need;
    if (whole || lo == hi) break;
    __syncthreads();  // (bins and pick are written again)
  }
  // Taken: keys from `lowest` on, and where not all of [lo, hi] are, which is one key then,
  // the first `need` of those.
  const uint32_t lowest = whole ? lo : hi + 1;
  if (!counted) {
    uint32_t n_over = 0, n_same = 0;
    each([&](int, const uint32_t (&key)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        n_over += __popcll(__ballot(key[c] > hi));
        n_same += __popcll(__ballot(key[c] - lo <= hi - lo));
      }
    });
    if (lane == 0) s.part[3][wave] = n_over, s.part[4][wave] = n_same;
    __syncthreads();
    above += row_all_of(earlier ? s.part[3][other] : 0u, plus);
    ties += row_all_of(earlier ? s.part[4][other] : 0u, plus);
  }
  if (whole) above += ties;
  auto number = [&](auto put) {
    each([&](int turn, const uint32_t (&key)[4]) {
      const int at = begin + 256 * turn + 4 * lane;
      uint32_t to = above;
      uint64_t over[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        over[c] = __ballot(key[c] >= lowest);
        to = below(over[c], to);
        above += __popcll(over[c]);
      }
      if (whole) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (key[c] >= lowest) put(to, at + c);
          to += key[c] >= lowest;
        }
        return;
      }
      uint32_t tie = ties;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint64_t same = __ballot(key[c] == lo);
        tie = below(same, tie);
        ties += __popcll(same);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool is_over = key[c] >= lowest, is_same = key[c] == lo;
        if (is_over || (is_same && tie < need)) put(to + min(tie, need), at + c);
        to += is_over;
        tie += is_same;
      }
    });
  };
  if (count <= kBins) {  // through LDS, to be written side by side
    number([&](uint32_t to, int i) { s.bins[to] = (uint32_t)i; });
    __syncthreads();
    for (int i = tid; i < count; i += kThreads) out[i] = (int)s.bins[i];
  } else {
    number([&](uint32_t to, int i) { out[to] = i; });
  }
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
  const bool wide = aligned(scores, 16) && (rows == 1 || row_stride % 4 == 0);
  // Threads: a wave's own work (scans, barriers) is most of a short row's, so that fewer are
  // better for short rows and, once the chip is full, for longer ones, as long as two keys a
  // thread reach k (one row of 4,096, k = 512: 4.7 us with half of the threads, 6.3 with all;
  // 1,430 rows of 8,192, 512 of each: 18.2 and 21.6, 2,048 of each: 26.9 and 23.3).
  const bool half = k <= 1024 && (width <= 4096 || (rows >= 1024 && width <= 8192));
  const auto kern = width <= 2048    ? index_topk_kernel<256, 2, false>
                    : half           ? width <= 4096 ? index_topk_kernel<512, 2, false>
                                                     : index_topk_kernel<512, 4, false>
                    : width <= 8192  ? index_topk_kernel<1024, 2, false>
                    : width <= 16384 ? index_topk_kernel<1024, 4, false>
                    : width <= 32768 ? index_topk_kernel<1024, 8, false>
                                     : index_topk_kernel<1024, 8, true>;
  const int threads = width <= 2048 ? 256 : half ? 512 : 1024;
  // A launch has fewer than 2^32 threads: with more the count wraps, without an error.
  constexpr int64_t kLaunchRows = (int64_t)1 << 21;
  for (int64_t at = 0; at < rows; at += kLaunchRows) {
    const TopkArgs a{scores ? scores + at * row_stride : nullptr, row_stride,
                     lengths ? lengths + at : nullptr, (int)width, (int)k, wide,
                     indices ? indices + at * k : nullptr, counts + at};
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min(rows - at, kLaunchRows)), dim3(threads), 0,
                       (hipStream_t)stream, a);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  return RM_OK;
}
