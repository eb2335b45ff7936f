// Attention of drafted trees over Native rows. Node j of request b, at depth d (0 for the
// children of the committed text), stands at position p = length + d; it sees the
// committed rows p - window + 1 .. length - 1, the nodes on its path and itself (as far as
// the window goes), and the compressed records of the history, if there are any. For each
// head: l_r = (q . K_r) * scale over the rows r that it sees, Z = sum exp(l_r) + exp(sink),
// out = sum exp(l_r) K_r / Z, lse = ln Z.
//
// All nodes and heads of a request read the same rows: row m = node * heads + head of q is
// one of its nodes * heads query rows. A workgroup takes 32 of them and a share of the
// request's rows, 128 a round: eight units of 16, one a wave. In a round a wave
//   * copies its unit of the next round to LDS as it is stored (global_load_lds),
//   * scores its unit: S^T = K Q^T on v_mfma_f32_16x16x32_bf16 for both halves of the 32
//     query rows, Q in registers, the codes made BF16 with their scales on the way from LDS
//     (the conversion's operand), and leaves the weights P^T = 2^(s - m) in LDS,
//   * adds all eight units to the 64 output coordinates that it owns: O^T += V^T P^T. V^T
//     comes out of LDS transposed (ds_read_b64_tr_b8), and P^T as the lanes left it: the
//     order of the rows in that product's long axis is free, and S^T's is taken. The codes
//     become BF16 without their scales there: a row's scale is a power of two, so it goes
//     to the weights' exponents, and as the eight waves own one group of 64 coordinates
//     each, once a weight and wave. Weights stand as P * 2^127 in BF16, and
//     (254 - scale byte) << 7 is subtracted as integers, saturating at zero: exact for
//     every byte but 255, whose row has NaN scores; what falls below 2^-126 becomes zero.
// Two barriers a round: before the copies (everyone is done with the buffer) and between
// weights and values. m is a whole number of log2 units, kept 16 above the largest score of
// the round that set it, so that it hardly ever moves again; a unit with a score above it
// takes its own for that round, and the waves then agree on the highest: integer
// subtractions on the weights' exponents, O rescaled and one barrier more.
// The output is divided by the sum of the weights as they were rounded, and lse takes the
// sum of the exact ones: roundings that a row's weights have in common cancel.
//
// LDS holds a row's 36 pieces of 16 bytes in a row, with the order in each four of them
// turned by the row's number (the copies choose their source), so that eight lanes reading
// one piece of eight rows meet every bank once.
//
// Units that some node does not see whole (the ends of the window and of the committed
// rows, the drafted rows) are masked by row; rows there that nobody sees, and rows with
// an infinity or NaN, are set to zero, the latter's scores to NaN where they are seen: a
// zero weight must not meet them.
#include <algorithm>

#include "combine.h"
#include "lds.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kWaves = 8;
constexpr int kRows = 32;  // query rows of a workgroup
constexpr int kUnit = 16;  // rows a wave scores in a round
constexpr int kRound = kWaves * kUnit;
constexpr int kMaxNodes = 64;
constexpr int kMaxHeads = 1024;
constexpr int kUnitBytes = kUnit * kNativeDataBytes;  // 9,216
constexpr int kCopies = kUnitBytes / 1024;            // 9
constexpr int kWeightsAt = 2 * kWaves * kUnitBytes;   // [4 pairs of units][2][64 lanes] 16 bytes
constexpr int kShiftsAt = kWeightsAt + 8 * 1024;      // [4][8 groups][4][8] u16
constexpr int kRefsAt = kShiftsAt + 4 * 8 * 64;       // [8 units][32 query rows] float
constexpr int kMovedAt = kRefsAt + kWaves * kRows * 4;  // [2]
constexpr int kLdsBytes = kMovedAt + 16;
constexpr int kSumsAt = kWeightsAt;  // at the end: [8 waves][32] of l, r
static_assert(kLdsBytes <= 160 * 1024 && kCopies * 1024 == kUnitBytes, "LDS of a CU");
constexpr float kHeadroom = 16.0f;

struct TreeArgs {
  const uint16_t* q;
  int nodes, heads;
  int q_rows;  // nodes * heads
  int tiles;   // of 32 of them
  const uint8_t* pool;
  int pool_pages;
  const int32_t* table;
  int64_t table_stride;
  int blocks;
  const int32_t* lengths;
  const int32_t* parents;
  int window;  // 0x7fffffff: none
  const uint8_t* past;  // the compressed records
  int past_pages;
  const int32_t* past_table;
  int64_t past_stride;
  int past_blocks;
  const int32_t* past_lengths;
  const float* sink;
  float scale_log2;
  int splits;
  uint16_t* out;
  float* lse;
  float* ws_o;  // null: one split, finish in place
  float* ws_lse;
};

__device__ __forceinline__ uint32_t from_lane(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * lane, (int)x);
}
// Nonzero where one of the dword's four E4M3 codes is NaN (0x7f or 0xff), or one of its two
// BF16 an infinity or NaN.
__device__ __forceinline__ uint32_t special(uint32_t x, bool bf16) {
  return ((x & (bf16 ? 0x7f807f80u : 0x7f7f7f7fu)) + (bf16 ? 0x00800080u : 0x01010101u)) &
         (bf16 ? 0x80008000u : 0x80808080u);
}
// Eight codes times a scale -> eight BF16.
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi, float scale) {
  return as_bf16x8(u32x4{fp8_pair_to_bf16<false>(lo, scale), fp8_pair_to_bf16<true>(lo, scale),
                         fp8_pair_to_bf16<false>(hi, scale), fp8_pair_to_bf16<true>(hi, scale)});
}

// Over the four lanes that share lane % 16.
__device__ __forceinline__ float over_groups(float x, bool is_max) {
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = is_max ? fmaxf(u2f(a[0]), u2f(a[1])) : u2f(a[0]) + u2f(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return is_max ? fmaxf(u2f(b[0]), u2f(b[1])) : u2f(b[0]) + u2f(b[1]);
}

struct Tree {
  const TreeArgs& a;
  const uint32_t lds;
  int lane, row, group;
  const int wave, b;
  // the request
  int held, past, first, past_units, units;
  // by half of the query rows, lane % 16: what the row's node sees, and its softmax
  bool live[2];
  int lowest[2];  // committed position
  uint32_t path[2][2];
  float m[2], l[2], r[2];
  u32x4 q[2][16];
  f32x4 o[2][4];  // coordinates 64 wave + 16 u + 4 group + i

  __device__ __forceinline__ Tree(const TreeArgs& args, uint32_t at, int request)
      : a(args),
        lds(at),
        lane(wave_lane()),
        row(lane & 15),
        group(lane >> 4),
        wave(uniform((int)(threadIdx.x >> 6))),
        b(request) {}

  // What follows from the lane is worked out again in each round: kept, it would push Q out
  // of the registers.
  __device__ __forceinline__ void again() {
    asm volatile("" : "+v"(lane));
    row = lane & 15;
    group = lane >> 4;
  }

  // Coordinates 64 s + 16 group .. + 15 as two operands, then the tail's 32 t + 8 group.
  __device__ __forceinline__ void load_q(int first_row) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int at = min(first_row + 16 * c + row, a.q_rows - 1);
      const uint16_t* const from = a.q + ((int64_t)b * a.q_rows + at) * kHeadDim;
#pragma unroll
      for (int s = 0; s < 7; ++s) {
        q[c][2 * s] = *(const u32x4*)(from + 64 * s + 16 * group);
        q[c][2 * s + 1] = *(const u32x4*)(from + 64 * s + 16 * group + 8);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
        q[c][14 + t] = *(const u32x4*)(from + kNopeDim + 32 * t + 8 * group);
    }
  }

  __device__ __forceinline__ void request() {
    held = max(min(a.lengths[b], 0x7fffff00), 0);
    past = 0;
    if (a.past_lengths) past = max(min(a.past_lengths[b], a.past_blocks * kPageRecords), 0);
    first = max(held - a.window + 1, 0) & ~(kUnit - 1);
    const int end = (int)min((int64_t)held + a.nodes, (int64_t)a.blocks * kPageRecords);
    past_units = (past + kUnit - 1) / kUnit;
    units = past_units + max((end - first + kUnit - 1) / kUnit, 0);
  }

  // Lane j works out node j's path; each lane then takes its query rows' nodes.
  __device__ __forceinline__ void tree(int first_row) {
    int up = -1;
    bool bad = lane >= a.nodes;
    if (!bad) {
      const int p = a.parents[(int64_t)b * a.nodes + lane];
      bad = p < -1 || p >= lane;
      up = bad ? -1 : p;
    }
    uint64_t seen = 1ull << lane;
    // twice as many steps up each time
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const int at = max(up, 0);
      const uint32_t lo = from_lane((uint32_t)seen, at), hi = from_lane((uint32_t)(seen >> 32), at);
      const uint32_t bad_up = from_lane(bad, at);
      const int up_up = (int)from_lane((uint32_t)up, at);
      if (up >= 0) {
        seen |= (uint64_t)hi << 32 | lo;
        bad = bad || bad_up;
        up = up_up;
      }
    }
    const int depth = __popcll(seen) - 1;
    // ancestors before the window (a path's nodes are in the order of their numbers)
    for (int n = depth + 1; n > a.window; --n) seen &= seen - 1;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int at = first_row + 16 * c + row;
      const int node = min(at / a.heads, a.nodes - 1);
      const uint32_t padding = from_lane(bad, node);  // (every lane takes part)
      live[c] = at < a.q_rows && !padding;
      path[c][0] = from_lane((uint32_t)seen, node);
      path[c][1] = from_lane((uint32_t)(seen >> 32), node);
      lowest[c] = held + (int)from_lane((uint32_t)depth, node) - a.window + 1;
    }
  }

  // Number of the page that unit i of the request lies in.
  __device__ __forceinline__ int page_of(int i) const {
    const bool of_past = i < past_units;
    const int at = of_past ? i * kUnit : first + (i - past_units) * kUnit;
    return of_past ? a.past_table[b * a.past_stride + at / kPageRecords]
                   : a.table[b * a.table_stride + at / kPageRecords];
  }
  struct Unit {
    const uint8_t* rows;  // of the page: the unit's data
    int at;               // its first record or position
    bool past, mapped;
    u32x2 scales;  // of row lane % 16
  };
  __device__ __forceinline__ Unit unit(int i, int page) const {
    Unit x;
    x.past = i < past_units;
    x.at = x.past ? i * kUnit : first + (i - past_units) * kUnit;
    page = uniform(page);
    x.mapped = page >= 0 && page < (x.past ? a.past_pages : a.pool_pages);
    const uint8_t* const from =
        (x.past ? a.past : a.pool) + (int64_t)(x.mapped ? page : 0) * kNativePageBytes;
    const int at = x.at & (kPageRecords - 1);
    x.rows = from + at * kNativeDataBytes;
    x.scales = *(const u32x2*)(from + kPageRecords * kNativeDataBytes + (at + row) * kScaleBytes);
    return x;
  }
  // Whether every live query row sees all of the unit.
  __device__ __forceinline__ bool whole(const Unit& x) const {
    return x.mapped && (x.past ? x.at + kUnit <= past
                               : x.at + kUnit <= held && x.at >= held + a.nodes - a.window);
  }
  // Piece j of row r goes to place j ^ turn(r) of the row, within its four.
  __device__ __forceinline__ static int turn(int r) { return (r >> 1) & 3; }
  __device__ __forceinline__ void copy(const Unit& x, uint32_t to) const {
#pragma unroll
    for (int n = 0; n < kCopies; ++n) {
      const uint32_t p = 64 * n + lane, r = p / 36, j = p - 36 * r;
      copy16(x.rows + (576 * r + 16 * (j ^ turn(r))), to + 1024 * n);
    }
  }

  // Where the lane leaves the weights of the wave's unit.
  __device__ __forceinline__ uint32_t weights_at(int c) const {
    return lds + kWeightsAt + 2048 * (wave >> 1) + 1024 * c + 16 * lane + 8 * (wave & 1);
  }
  // Scores and weights of the unit, in LDS at `at`.
  template <bool kWhole>
  __device__ __forceinline__ void score(const Unit& x, uint32_t at, float (&own)[2], float (&sum)[2],
                                        float (&rsum)[2]) {
    u32x2 bytes = x.scales;
    // rows of the unit that count
    const int stop = min(x.past ? past - x.at : held + a.nodes - x.at, kUnit);
    uint32_t odd = 0;  // rows with an infinity or NaN
    if (!kWhole) {
      // row `row`, pieces 9 group .. + 8: an infinity or NaN in it?
      const uint32_t mine = at + kNativeDataBytes * row + 144 * group;
      uint32_t bad = 0;
#pragma unroll
      for (int n = 0; n < 9; ++n) {
        const u32x4 v = lds_read<u32x4>(mine + 16 * n);
        // (pieces 28 and up are the tail)
        const bool tail = 9 * group + n >= 28;
#pragma unroll
        for (int k = 0; k < 4; ++k) bad |= special(v[k], tail);
      }
#pragma unroll
      for (int g = 0; g < 7; ++g)
        bad |= ((bytes[g / 4] >> (8 * (g % 4))) & 0xffu) == 0xffu;
      const uint64_t found = __ballot(bad != 0);
      odd = (uint32_t)(found | found >> 16 | found >> 32 | found >> 48) & 0xffffu;
      if (!x.mapped || row >= stop || ((odd >> row) & 1u)) {
#pragma unroll
        for (int n = 0; n < 9; ++n) lds_write(mine + 16 * n, u32x4{0, 0, 0, 0});
        bytes = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
      }
    }
    // shifts of row `row` for groups 2 group and 2 group + 1
    {
      const uint32_t two = (group >= 2 ? bytes[1] : bytes[0]) >> (16 * (group & 1));
      const uint32_t to = lds + kShiftsAt + 512 * (wave >> 1) + 128 * group + 16 * (row >> 2) +
                          2 * (4 * (wave & 1) + (row & 3));
      lds_write<uint16_t>(to, (uint16_t)((254u - (two & 0xffu)) << 7));
      lds_write<uint16_t>(to + 64, (uint16_t)((254u - ((two >> 8) & 0xffu)) << 7));
    }
    if (!kWhole) wave_lds_sync();
    f32x4 acc[2][2] = {};
    const uint32_t k_at = at + kNativeDataBytes * row + 16 * (group ^ turn(row));
#pragma unroll
    for (int s = 0; s < 7; ++s) {
      const float f = u2f(((bytes[s / 4] >> (8 * (s % 4))) & 0xffu) << 23);
      const u32x4 v = lds_read<u32x4>(k_at + 64 * s);
      const bf16x8 k0 = codes8(v[0], v[1], f), k1 = codes8(v[2], v[3], f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        acc[c][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, as_bf16x8(q[c][2 * s]), acc[c][0],
                                                            0, 0, 0);
        acc[c][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, as_bf16x8(q[c][2 * s + 1]),
                                                            acc[c][1], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bf16x8 k = as_bf16x8(lds_read<u32x4>(k_at + kNopeDim + 64 * t));
#pragma unroll
      for (int c = 0; c < 2; ++c)
        acc[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, as_bf16x8(q[c][14 + t]), acc[c][t],
                                                            0, 0, 0);
    }
    // value i is row 4 group + i of the unit
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f32x4 s = (acc[c][0] + acc[c][1]) * a.scale_log2;
      if (!kWhole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 4 * group + i, p = x.at + n, node = p - held;
          const uint32_t word = node < 32 ? path[c][0] : path[c][1];
          const bool on_path = ((word >> (node & 31)) & 1u) != 0;
          const bool see = live[c] & x.mapped & (n < stop) &
                           (x.past | (node < 0 ? p >= lowest[c] : on_path));
          s[i] = (odd >> n) & 1u ? NAN : s[i];
          s[i] = see ? s[i] : -INFINITY;
        }
      }
      const float top = over_groups(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), true);
      own[c] = top > m[c] ? ceilf(top) + kHeadroom : m[c];
      const float ref = own[c] == -INFINITY ? 0.0f : own[c];
      f32x4 p;
      sum[c] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = __builtin_amdgcn_exp2f(s[i] - ref);
        sum[c] += p[i];
        p[i] *= 0x1p127f;
      }
      const u32x2 d = {__builtin_bit_cast(uint32_t, bf16_pair(p[0], p[1])),
                       __builtin_bit_cast(uint32_t, bf16_pair(p[2], p[3]))};
      rsum[c] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rsum[c] = __builtin_fmaf(i & 1 ? u2f(d[i / 2] & 0xffff0000u) : u2f(d[i / 2] << 16),
                                 0x1p-127f, rsum[c]);
      lds_write(weights_at(c), d);
    }
  }

  // O += the round's units, at `at`.
  __device__ __forceinline__ void add(uint32_t at) {
    const bool tail = wave == kWaves - 1;  // the BF16 coordinates
    const int pair = row >> 1;  // transposed reads: row 4 group + pair % 4 of unit pair / 4
    const int of = 4 * group + (pair & 3);
    const uint32_t v_at = at + kUnitBytes * (pair >> 2) + kNativeDataBytes * of + 64 * wave +
                          8 * (row & 1);
    const int tail_of = 4 * group + (row >> 2);
    const uint32_t t_at = at + kNativeDataBytes * tail_of + kNopeDim + 8 * (row & 1);
#pragma unroll
    for (int v = 0; v < kWaves / 2; ++v) {
      u32x4 p[2], shift = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};  // 127 << 7
      bf16x8 x[4];
      if (!tail) {
        shift = lds_read<u32x4>(lds + kShiftsAt + 512 * v + 64 * wave + 16 * group);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const i32x2 codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(lds_void*)(
              uintptr_t)(v_at + 16 * (u ^ turn(of)) + 2 * kUnitBytes * v));
          x[u] = codes8((uint32_t)codes[0], (uint32_t)codes[1], 1.0f);
        }
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          u32x2 part[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)  // pieces 28 + 2 u and + 1
            part[k] = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)(uintptr_t)(
                           t_at + kUnitBytes * (2 * v + k) + 64 * (u >> 1) +
                           16 * ((2 * (u & 1) + ((row & 3) >> 1)) ^ turn(tail_of)))));
          x[u] = as_bf16x8(u32x4{part[0][0], part[0][1], part[1][0], part[1][1]});
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        p[c] = lds_read<u32x4>(lds + kWeightsAt + 2048 * v + 1024 * c + 16 * lane);
#pragma unroll
        for (int k = 0; k < 4; ++k) p[c][k] = sub_sat(p[c][k], shift[k]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          o[c][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u], as_bf16x8(p[c]), o[c][u], 0, 0, 0);
    }
  }

  // Units [begin, end).
  __device__ __forceinline__ void run(int begin, int end) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[c] = -INFINITY;
      l[c] = r[c] = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[c][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (threadIdx.x == 0) lds_write(lds + kMovedAt, u32x2{0, 0});
    Unit x{}, next{};
    int page = 0;
    if (begin + wave < end) {
      x = unit(begin + wave, page_of(begin + wave));
      copy(x, lds + wave * kUnitBytes);
    }
    if (begin + kWaves + wave < end) page = page_of(begin + kWaves + wave);
    int odd = 0;  // round
    for (int i = begin + wave; i - wave < end; i += kWaves, odd ^= 1) {
      const uint32_t at = lds + odd * kWaves * kUnitBytes;
      again();
      wait_copies<0>();
      lds_barrier();
      if (i + kWaves < end) {
        next = unit(i + kWaves, page);
        copy(next, lds + (odd ^ 1) * kWaves * kUnitBytes + wave * kUnitBytes);
        if (i + 2 * kWaves < end) page = page_of(i + 2 * kWaves);
      }
      float own[2] = {m[0], m[1]}, sum[2] = {0.f, 0.f}, rsum[2] = {0.f, 0.f};
      const uint32_t mine = at + wave * kUnitBytes;
      if (i < end) {
        if (whole(x))
          score<true>(x, mine, own, sum, rsum);
        else
          score<false>(x, mine, own, sum, rsum);
      } else {  // the round's last units: nothing
#pragma unroll
        for (int n = 0; n < kCopies; ++n) lds_write(mine + 1024 * n + 16 * lane, u32x4{0, 0, 0, 0});
#pragma unroll
        for (int c = 0; c < 2; ++c) lds_write(weights_at(c), u32x2{0, 0});
      }
      if (lane < kUnit) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
          lds_write(lds + kRefsAt + 4 * (kRows * wave + 16 * c + row), own[c]);
      }
      if (__ballot(own[0] != m[0] || own[1] != m[1]) != 0 && lane == 0)
        lds_write(lds + kMovedAt + 4 * odd, 1);
      if (threadIdx.x == 0) lds_write(lds + kMovedAt + 4 * (odd ^ 1), 0);
      lds_barrier();
      if (uniform(lds_read<int>(lds + kMovedAt + 4 * odd)) != 0) {
        // the highest reference is everyone's: O, the sums and the unit's weights go down to it
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = m[c];
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            top = fmaxf(top, lds_read<float>(lds + kRefsAt + 4 * (kRows * w + 16 * c + row)));
          // (equal ones may both be infinite)
          const float f = m[c] == top ? 1.0f : __builtin_amdgcn_exp2f(m[c] - top);
          const float g = own[c] == top ? 1.0f : __builtin_amdgcn_exp2f(own[c] - top);
          m[c] = top;
          l[c] *= f;
          r[c] *= f;
          sum[c] *= g;
          rsum[c] *= g;
#pragma unroll
          for (int u = 0; u < 4; ++u) o[c][u] *= f;
          // whole log2 units, in both exponents; 255: past every exponent, also for a
          // difference that is NaN (infinities: the sum is NaN then)
          const uint32_t down = __umul24((uint32_t)fminf(top - own[c], 255.0f), 0x00800080u);
          const u32x2 p = lds_read<u32x2>(weights_at(c));
          lds_write(weights_at(c), u32x2{sub_sat(p[0], down), sub_sat(p[1], down)});
        }
        lds_barrier();
      }
      again();
#pragma unroll
      for (int c = 0; c < 2; ++c) l[c] += sum[c], r[c] += rsum[c];
      add(at);
      x = next;
    }
  }

  __device__ __forceinline__ void finish(int first_row, int split) {
    lds_barrier();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[c] = over_groups(l[c], false);
      r[c] = over_groups(r[c], false);
      if (lane < 16) lds_write(lds + kSumsAt + 8 * (kRows * wave + 16 * c + row), f32x2{l[c], r[c]});
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = 0.0f, rsum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const f32x2 of = lds_read<f32x2>(lds + kSumsAt + 8 * (kRows * w + 16 * c + row));
        sum += of[0];
        rsum += of[1];
      }
      const int at = first_row + 16 * c + row;
      if (at >= a.q_rows) continue;
      if (!live[c]) sum = 0.0f;
      const int node = at / a.heads, h = at - node * a.heads;
      const int64_t token = (int64_t)b * a.nodes + node;
      const int c0 = 64 * wave + 4 * group;
      if (a.ws_o) {
        const int64_t to = (token * a.splits + split) * a.heads + h;
        const float f = sum != 0.0f ? 1.0f / rsum : 0.0f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          f32x4 x = o[c][u] * f;
          if (sum == 0.0f) x = f32x4{0.f, 0.f, 0.f, 0.f};
          __builtin_nontemporal_store(x, (f32x4*)(a.ws_o + to * kHeadDim + c0 + 16 * u));
        }
        // (NaN goes on as infinity: the combine's maximum would pass over a NaN)
        if (wave == 0 && group == 0)
          a.ws_lse[to] = sum != sum     ? INFINITY
                         : sum != 0.0f ? m[c] + __builtin_amdgcn_logf(sum)
                                       : -INFINITY;
        continue;
      }
      const float sink2 = a.sink ? a.sink[h] * kLog2e : -INFINITY;
      const float top = fmaxf(sum != 0.0f ? m[c] : -INFINITY, sink2);
      float f = 0.0f, lse = -INFINITY;
      if (top != -INFINITY || sum != 0.0f) {
        const float em = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[c] - top);
        const float z = sum * em + __builtin_amdgcn_exp2f(sink2 - top);
        // (O over the rounded weights' sum, times the rows' share of Z)
        if (sum != 0.0f) f = sum * em / (rsum * z);
        lse = (top + __builtin_amdgcn_logf(z)) * kLn2;
      }
      if (wave == 0 && group == 0) a.lse[token * a.heads + h] = lse;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 x = o[c][u] * f;
        if (sum == 0.0f) x = f32x4{0.f, 0.f, 0.f, 0.f};
        *(u32x2*)(a.out + (token * a.heads + h) * kHeadDim + c0 + 16 * u) =
            u32x2{__builtin_bit_cast(uint32_t, bf16_pair(x[0], x[1])),
                  __builtin_bit_cast(uint32_t, bf16_pair(x[2], x[3]))};
      }
    }
  }
};

__global__ __launch_bounds__(64 * kWaves, 2) void tree_decode_kernel(TreeArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLdsBytes];
  const int b = (int)blockIdx.x / a.tiles;
  const int first_row = ((int)blockIdx.x - b * a.tiles) * kRows;
  const int split = (int)blockIdx.y;
  Tree t(a, (uint32_t)(uintptr_t)(lds_void*)lds, b);
  t.load_q(first_row);
  t.request();
  t.tree(first_row);
  const int share = ((t.units + a.splits - 1) / a.splits + kWaves - 1) / kWaves * kWaves;
  const int begin = min(split * share, t.units);
  t.run(begin, min(begin + share, t.units));
  t.finish(first_row, split);
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

bool bad_sizes(int64_t batch, int64_t nodes, int64_t heads, int64_t blocks, int64_t window,
               int64_t past_blocks) {
  return batch < 0 || nodes < 0 || nodes > kMaxNodes || heads < 0 || heads > kMaxHeads ||
         batch > 65535 || batch * nodes > 65535 || blocks < 0 || blocks > (1 << 24) ||
         window < 0 || window > 0x7fffffff || past_blocks < 0 || past_blocks > (1 << 24);
}

int plan(int64_t batch, int64_t nodes, int64_t heads, int64_t blocks, int64_t window,
         int64_t past_blocks) {
  const int64_t tiles = std::max<int64_t>(batch * ((nodes * heads + kRows - 1) / kRows), 1);
  int64_t rows = blocks * kPageRecords;
  if (window > 0) rows = std::min(rows, window + nodes + kUnit);
  const int64_t rounds = (rows + past_blocks * kPageRecords + kRound - 1) / kRound;
  const int64_t most = std::min<int64_t>({256 / tiles, rounds, kMaxSplits});
  return (int)std::max<int64_t>(most, 1);
}
size_t ws_bytes(int64_t splits, int64_t rows) {
  return splits > 1 ? (size_t)(splits * rows) * (kHeadDim + 1) * sizeof(float) : 0;
}

}  // namespace

extern "C" int rm_tree_decode_workspace(int64_t batch, int64_t nodes, int64_t heads,
                                        int64_t max_blocks, int64_t window, int64_t history_blocks,
                                        int32_t* num_splits, size_t* workspace_bytes) {
  if (bad_sizes(batch, nodes, heads, max_blocks, window, history_blocks)) return RM_ERR_SHAPE;
  const int splits = plan(batch, nodes, heads, max_blocks, window, history_blocks);
  if (num_splits) *num_splits = splits;
  if (workspace_bytes) *workspace_bytes = ws_bytes(splits, batch * nodes * heads);
  return RM_OK;
}

extern "C" int rm_tree_decode_fwd(const uint16_t* q, int64_t batch, int64_t nodes, int64_t heads,
                                  const uint8_t* pool, int64_t pool_pages,
                                  const int32_t* block_table, int64_t block_table_stride,
                                  int64_t max_blocks, const int32_t* lengths,
                                  const int32_t* parents, int64_t window,
                                  const uint8_t* history_pool, int64_t history_pages,
                                  const int32_t* history_table, int64_t history_table_stride,
                                  int64_t history_blocks, const int32_t* history_lengths,
                                  const float* sink, float softmax_scale, uint16_t* out, float* lse,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_sizes(batch, nodes, heads, max_blocks, window, history_blocks) || pool_pages < 0 ||
      pool_pages > ((int64_t)1 << 25) || history_pages < 0 ||
      history_pages > ((int64_t)1 << 25) || block_table_stride < max_blocks ||
      history_table_stride < history_blocks)
    return RM_ERR_SHAPE;
  if (batch == 0 || nodes == 0 || heads == 0) return RM_OK;
  if (!q || !out || !lse || !lengths || !parents ||
      (max_blocks > 0 && (!block_table || (pool_pages > 0 && !pool))) ||
      (history_blocks > 0 &&
       (!history_table || !history_lengths || (history_pages > 0 && !history_pool))))
    return RM_ERR_NULL;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(pool, 16) || !aligned(history_pool, 16))
    return RM_ERR_ALIGN;
  for (const void* p : {(const void*)block_table, (const void*)lengths, (const void*)parents,
                        (const void*)history_table, (const void*)history_lengths,
                        (const void*)sink, (const void*)lse})
    if (!aligned(p, 4)) return RM_ERR_ALIGN;
  const int64_t rows = batch * nodes * heads;
  const int splits = plan(batch, nodes, heads, max_blocks, window, history_blocks);
  const size_t bytes = ws_bytes(splits, rows);
  if (bytes > 0 && (!workspace || workspace_bytes < bytes)) return RM_ERR_WORKSPACE;
  if (bytes > 0 && !aligned(workspace, 16)) return RM_ERR_ALIGN;
  TreeArgs a;
  a.q = q;
  a.nodes = (int)nodes;
  a.heads = (int)heads;
  a.q_rows = (int)(nodes * heads);
  a.tiles = (a.q_rows + kRows - 1) / kRows;
  a.pool = pool;
  a.pool_pages = (int)pool_pages;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.blocks = pool_pages > 0 ? (int)max_blocks : 0;
  a.lengths = lengths;
  a.parents = parents;
  a.window = window > 0 ? (int)window : 0x7fffffff;
  a.past = history_pool;
  a.past_pages = (int)history_pages;
  a.past_table = history_table;
  a.past_stride = history_table_stride;
  a.past_blocks = (int)history_blocks;
  a.past_lengths = history_blocks > 0 && history_pages > 0 ? history_lengths : nullptr;
  a.sink = sink;
  a.scale_log2 = softmax_scale * kLog2e;
  a.splits = splits;
  a.out = out;
  a.lse = lse;
  a.ws_o = splits > 1 ? (float*)workspace : nullptr;
  a.ws_lse = splits > 1 ? (float*)workspace + (size_t)splits * rows * kHeadDim : nullptr;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(tree_decode_kernel, dim3((unsigned)(batch * a.tiles), (unsigned)splits),
                     dim3(64 * kWaves), 0, s, a);
  if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  if (splits > 1) {
    launch_combine<true>(a.ws_o, a.ws_lse, sink, splits, batch * nodes, heads, out, lse, s);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  return RM_OK;
}
