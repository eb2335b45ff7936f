// Attention of drafted trees over Native rows. Node j of request b, at depth d (0 for the
// children of the committed text), stands at position p = length + d; it sees the
// committed rows p - window + 1 .. length - 1, the nodes on its path and itself (as far as
// the window goes), and the compressed records of the history, if there are any. For each
// head: l_r = (q . K_r) * scale over the rows r that it sees, Z = sum exp(l_r) + exp(sink),
// out = sum exp(l_r) K_r / Z, lse = ln Z.
//
// All nodes and heads of a request read the same rows: row m = node * heads + head of q is
// one of its nodes * heads query rows. A workgroup takes 32 of them and a share of the
// request's rows, 64 a round: four units of 16. Eight waves, two a SIMD, in two roles, so
// that one's vector work and waits lie under the other's matrix products:
//   * four scorers, each with all 32 query rows (Q in registers) and a unit of the round:
//     S^T = K Q^T on v_mfma_f32_16x16x32_bf16, the codes made BF16 with their scales on the
//     way from LDS (the conversion's operand), once for both halves of the query rows; they
//     leave the weights P^T = 2^(s - m) in LDS;
//   * four adders, each with 128 output coordinates of all 32 query rows (in registers):
//     O^T += V^T P^T of the round before. V^T comes out of LDS transposed
//     (ds_read_b64_tr_b8), and P^T as the scorers left it: the order of the rows in that
//     product's long axis is free, and S^T's is taken. The codes become BF16 without their
//     scales there: a row's scale is a power of two, so it goes to the weights' exponents,
//     and as an adder owns two groups of 64 coordinates each, twice a weight and wave.
//     Weights stand as P * 2^127 in BF16, and (254 - scale byte) << 7 is subtracted as
//     integers, saturating at zero: exact for every byte but 255, whose row has NaN scores;
//     what falls below 2^-126 becomes zero. The adders also copy the rows of the round after
//     next to LDS as they are stored (global_load_lds), while a round's operands come.
// One barrier a round. m is a whole number of log2 units, kept 16 above the largest score of
// the round that set it, so that it hardly ever moves again; a unit with a score above it
// takes its own for that round. After it the scorers go on from the highest of the units',
// and the adders lower that round's weights (integer subtractions on their exponents) and O.
// The output is divided by the sum of the weights as they were rounded, and lse takes the
// sum of the exact ones: roundings that a row's weights have in common cancel. The weights are
// the one thing held in fewer bits, as the matrix instruction takes them: outputs are up to
// 0.0020 off, 0.0017 by their own rounding to BF16.
//
// LDS holds a row's 36 pieces of 16 bytes in a row, with the order in each four of them
// turned by the row's number (the copies choose their source), so that eight lanes reading
// one piece of eight rows meet every bank once.
//
// Bound by the two roles' waits for each other, one barrier a round: a round is 1,024 cycles of
// matrix instructions a SIMD and about 1,600 of vector ones (480 convert codes), and takes
// 1.35 us, some 3,200 cycles; vector issue takes 49 % of all cycles, the matrix pipes are
// busy in 32 % (16 requests of 256 query rows, 4,096 to 16,384 records: 117 us, 640 TFLOP/s; a
// large product reaches 1,189). 32 query rows, as the queries and outputs of more do not fit the
// registers of two waves a SIMD; 64 rows a round, as four rounds fill LDS. Small calls are
// their start and end: 8 x 16 query rows over 8,192 records take 18.4 us, of which three
// rounds are 4, the combine 4 and the launches 5.
//
// The rounds of all requests are dealt out evenly (deal()): 16 ragged requests 200 us with
// each request in two halves, 138 so.
//
// Units that some node does not see whole (the ends of the window and of the committed
// rows, the drafted rows) are masked by row; the adders take zeros for rows there that nobody
// sees, and for rows with an infinity or NaN, whose scores are NaN where they are seen: a
// zero weight must not meet them. Such rows are looked for only if a score is not finite.
#include <algorithm>
#include <cmath>

#include "combine.h"
#include "lds.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kRows = 32;    // query rows of a workgroup
constexpr int kUnit = 16;    // rows a scorer takes in a round
constexpr int kUnits = 4;    // of a round
constexpr int kRound = kUnits * kUnit;
constexpr int kScorers = 4;  // unit `wave`
constexpr int kAdders = 4;   // coordinates 128 (wave - 4) ..
constexpr int kBuffers = 4;  // rounds in LDS: added, scored, two being copied
constexpr int kMaxNodes = 64;
constexpr int kMaxHeads = 1024;
constexpr int kUnitBytes = kUnit * kNativeDataBytes;  // 9,216: nine copies of 64 pieces
constexpr int kScalesAt = kUnits * kUnitBytes;  // the units' scale rows, 8 bytes each
constexpr int kRoundBytes = kScalesAt + kUnits * kUnit * kScaleBytes;
constexpr int kCopies = 10;  // an adder and round: a unit and its scales
// Of odd and even rounds:
constexpr int kWeightsAt = kBuffers * kRoundBytes;  // [2 pairs of units][2][64 lanes] 16 bytes
constexpr int kWeightsBytes = 4 * 1024;
constexpr int kShiftsAt = kWeightsAt + 2 * kWeightsBytes;  // [2][8 groups][4][8] u16
constexpr int kShiftsBytes = 2 * 8 * 64;
constexpr int kRefsAt = kShiftsAt + 2 * kShiftsBytes;  // [4 units][32 query rows] float
constexpr int kRefsBytes = kUnits * kRows * 4;
constexpr int kStateAt = kRefsAt + 2 * kRefsBytes;  // [4 units]: bits of rows left out, kMoved
constexpr int kSumsAt = kStateAt + 2 * 16;          // [4 units][32 query rows] of l, r
constexpr int kStartsAt = kSumsAt + kUnits * kRows * 8;  // [requests + 1]
constexpr int kQueriesAt = 3 * kRoundBytes;  // before a piece's fourth round is copied
constexpr int kMaxShared = 256;   // requests whose rounds are dealt out evenly
constexpr int kLdsBytes = kStartsAt + (kMaxShared + 1) * 4;
// What a piece costs beyond its rounds, in rounds (about 8 us at 1.35 a round; window trees
// 36.8 us with two, 35.3 with four, 34.6 with six, large ones the same).
constexpr int kOverhead = 6;
static_assert(kLdsBytes <= 160 * 1024, "LDS of a CU");
constexpr uint32_t kMoved = 1u << 16;  // the unit took references of its own
constexpr float kHeadroom = 16.0f;
constexpr float kUnit27 = 0x1p-100f;  // of weights times 2^127, for their sum times 2^27

typedef __attribute__((address_space(4))) int32_t const_i32;  // scalar loads

struct TreeArgs {
  const uint16_t* q;
  int batch;
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
  float scale_log2;  // not below zero
  bool negated;      // and q times -1
  int parts;   // workgroups that share the rounds of a tile's requests; 0: a request each
  bool each_eighth;  // an XCD takes every eighth part, not one after the other
  int slots;   // partials that a request can have
  uint16_t* out;
  float* lse;
  float* ws_o;
  float* ws_lse;
  int32_t* counts;  // [batch] partials of the request; 0: finished in place
};
typedef const __attribute__((address_space(4))) TreeArgs const_args;

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

// (NaN if either is: fmaxf first quiets both, an instruction each)
__device__ __forceinline__ float higher(float x, float y) {
  return __builtin_elementwise_maximum(x, y);
}
__device__ __forceinline__ float lower(float x, float y) {
  return __builtin_elementwise_minimum(x, y);
}
// Over the four lanes that share lane % 16.
__device__ __forceinline__ float over_groups(float x, bool is_max) {
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = is_max ? higher(u2f(a[0]), u2f(a[1])) : u2f(a[0]) + u2f(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return is_max ? higher(u2f(b[0]), u2f(b[1])) : u2f(b[0]) + u2f(b[1]);
}

// Copies memory -> LDS of 16 or 4 bytes a lane, from base + offset to lds + 16 or 4 lane. As
// assembly, because the compiler orders the builtin's writes to LDS by waits of its own: it
// waited for all copies in flight before each transposed read and at each barrier (16 x 16
// nodes 316 us with the builtin, 292 so, both then). wait_copies() and the barriers order
// them here. (s_nop 4: a base that a vector instruction wrote, as one that was spilled is, may
// be read five wait states later; the compiler counts them for its own instructions only.)
__device__ __forceinline__ void copy_ahead16(const uint8_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(offset), "s"(base), "{m0}"(lds)
               : "memory");
}
// Four of them, each 1,024 bytes after the one before (an instruction's offset counts in both).
__device__ __forceinline__ void copy_ahead16x4(const uint8_t* base, uint32_t o0, uint32_t o1,
                                               uint32_t o2, uint32_t o3, uint32_t lds) {
  asm volatile(
      "s_nop 4\n\tglobal_load_lds_dwordx4 %0, %4\n\t"
      "global_load_lds_dwordx4 %1, %4 offset:%6\n\t"
      "global_load_lds_dwordx4 %2, %4 offset:%7\n\t"
      "global_load_lds_dwordx4 %3, %4 offset:%8"
      :
      : "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(base), "{m0}"(lds), "n"(1024), "n"(2 * 1024),
        "n"(3 * 1024)
      : "memory");
}
__device__ __forceinline__ void copy_ahead4(const uint8_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1"
               :
               : "v"(offset), "s"(base), "{m0}"(lds)
               : "memory");
}

// What both roles know.
struct Tree {
  const_args* a;
  const uint32_t lds;
  int lane, row, group;
  const int wave;
  int b;
  // the request: its rows of the block tables, and the pools (the compressed records first)
  const const_i32* table[2];
  const uint8_t* pool[2];
  int pages[2];
  int held, past, first, past_units, units;
  int begin, end;                            // the workgroup's units

  int slot, of_slots;                        // the piece among its request's

  __device__ __forceinline__ Tree(const_args* args, uint32_t at)
      : a(args),
        lds(at),
        lane(wave_lane()),
        row(lane & 15),
        group(lane >> 4),
        wave(uniform((int)(threadIdx.x >> 6))) {}

  struct Extent {
    int held, past, first, past_units, units;
  };
  __device__ __forceinline__ static Extent extent(const_args* a, int length, int past_length) {
    Extent x;
    x.held = max(min(length, 0x7fffff00), 0);
    x.past = max(min(past_length, a->past_blocks * kPageRecords), 0);
    x.first = max(x.held - a->window + 1, 0) & ~(kUnit - 1);
    const int stop = (int)min((int64_t)x.held + a->nodes, (int64_t)a->blocks * kPageRecords);
    x.past_units = (x.past + kUnit - 1) / kUnit;
    x.units = x.past_units + max((stop - x.first + kUnit - 1) / kUnit, 0);
    return x;
  }
  __device__ __forceinline__ static int rounds(const Extent& x) {
    return max((x.units + kUnits - 1) / kUnits, 1);
  }

  // Rounds from .. to - 1 of a request.
  __device__ __forceinline__ void piece(int request, int from, int to) {
    anew();
    b = request;
    const Extent x = extent(a, ((const const_i32*)a->lengths)[b],
                            a->past_lengths ? ((const const_i32*)a->past_lengths)[b] : 0);
    held = x.held, past = x.past, first = x.first, past_units = x.past_units, units = x.units;
    begin = min(from * kUnits, units);
    end = min(to, rounds(x)) * kUnits;
    end = min(end, units);
    table[0] = (const const_i32*)a->past_table + b * a->past_stride;
    table[1] = (const const_i32*)a->table + b * a->table_stride;
    pool[0] = a->past;
    pool[1] = a->pool;
    pages[0] = a->past_pages;
    pages[1] = a->pool_pages;
    // (kept in registers: chosen between in memory, each unit would wait for them again)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      asm volatile("" : "+s"(table[k]));
      asm volatile("" : "+s"(pool[k]));
      asm volatile("" : "+s"(pages[k]));
    }
  }
  // Number of the page that unit i of the request lies in.
  __device__ __forceinline__ int page_of(int i) const {
    const bool of_past = i < past_units;
    const int at = of_past ? i * kUnit : first + (i - past_units) * kUnit;
    return (of_past ? table[0] : table[1])[(uint32_t)at / kPageRecords];
  }
  // What follows from the lane is worked out again in each round: kept, it would push Q out
  // of the registers.
  __device__ __forceinline__ void anew() {
    asm volatile("" : "+s"(a));
    again();
  }
  __device__ __forceinline__ void again() {
    asm volatile("" : "+v"(lane));
    row = lane & 15;
    group = lane >> 4;
  }
  struct Unit {
    const uint8_t* page;
    int at;       // its first record or position
    int in_page;  // row there
    bool past, mapped;
  };
  __device__ __forceinline__ Unit unit(int i, int page) const {
    Unit x;
    x.past = i < past_units;
    x.at = x.past ? i * kUnit : first + (i - past_units) * kUnit;
    x.mapped = (uint32_t)page < (uint32_t)(x.past ? pages[0] : pages[1]);
    x.page = (x.past ? pool[0] : pool[1]) + (uint64_t)(x.mapped ? page : 0) * kNativePageBytes;
    x.in_page = x.at & (kPageRecords - 1);
    return x;
  }
  // Piece j of row r goes to place j ^ turn(r) of the row, within its four.
  __device__ __forceinline__ static int turn(int r) { return (r >> 1) & 3; }
  __device__ __forceinline__ uint32_t buffer(int round) const {
    return lds + (round & (kBuffers - 1)) * kRoundBytes;
  }
  __device__ __forceinline__ uint32_t ref_at(int round, int unit, int c) const {
    return lds + kRefsAt + (round & 1) * kRefsBytes + 4 * (kRows * unit + 16 * c + row);
  }
  // Of a round's units.
  __device__ __forceinline__ u32x4 state(int round) const {
    return lds_read<u32x4>(lds + kStateAt + 16 * (round & 1));
  }
};

// Unit `wave` of every round. By half c of the query rows, 16 c + lane % 16: what the row's
// node sees, and its softmax.
struct Scorer : Tree {
  const int of;
  bool live[2];
  int lowest[2];  // committed position
  uint32_t path[2][2];
  float m[2], l[2], r[2];
  float least;  // score of a whole unit
  u32x4 q[2][16];

  __device__ __forceinline__ Scorer(const Tree& t) : Tree(t), of(wave) {}

  // Rows 8 wave .. + 7 of Q to LDS. Piece j of row r goes to place j ^ (r & 15) there, so that
  // sixteen lanes reading one piece of sixteen rows meet every bank once.
  __device__ __forceinline__ void copy_q(int first_row) const {
    const uint8_t* const from =
        (const uint8_t*)(a->q + ((int64_t)b * a->q_rows + first_row) * kHeadDim);
#pragma unroll
    for (int n = 0; n < kRows / kScorers; ++n) {
      const int r = kRows / kScorers * of + n;
      copy_ahead16(from, 2 * kHeadDim * min(r, a->q_rows - 1 - first_row) + 16 * (lane ^ (r & 15)),
                   lds + kQueriesAt + 2 * kHeadDim * r);
    }
  }
  // Coordinates 64 s + 16 group .. + 15 as two operands, then the tail's 32 t + 8 group.
  __device__ __forceinline__ void load_q() {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t at = lds + kQueriesAt + 2 * kHeadDim * (16 * c + row);
#pragma unroll
      for (int s = 0; s < 14; ++s)
        q[c][s] = lds_read<u32x4>(at + 16 * ((8 * (s / 2) + 2 * group + (s & 1)) ^ row));
#pragma unroll
      for (int t = 0; t < 2; ++t)
        q[c][14 + t] = lds_read<u32x4>(at + 16 * ((56 + 4 * t + group) ^ row));
      if (a->negated) {
#pragma unroll
        for (int s = 0; s < 16; ++s) q[c][s] ^= 0x80008000u;
      }
    }
  }

  // Lane j works out node j's path (parent: of node lane); each lane then takes its query
  // row's node.
  __device__ __forceinline__ void tree(int first_row, int parent) {
    bool bad = lane >= a->nodes || parent < -1 || parent >= lane;
    int up = bad ? -1 : parent;
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
    for (int n = depth + 1; n > a->window; --n) seen &= seen - 1;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int at = first_row + 16 * c + row;
      const int node = min(at / a->heads, a->nodes - 1);
      const uint32_t padding = from_lane(bad, node);  // (every lane takes part)
      live[c] = at < a->q_rows && !padding;
      path[c][0] = from_lane((uint32_t)seen, node);
      path[c][1] = from_lane((uint32_t)(seen >> 32), node);
      lowest[c] = held + (int)from_lane((uint32_t)depth, node) - a->window + 1;
    }
  }

  // Whether every live query row sees all of the unit.
  __device__ __forceinline__ bool whole(const Unit& x) const {
    return x.mapped & (x.at + kUnit <= (x.past ? past : held)) &
           (x.past | (x.at >= held + a->nodes - a->window));
  }
  __device__ __forceinline__ uint32_t weights_at(int round, int c) const {
    return lds + kWeightsAt + (round & 1) * kWeightsBytes + 2048 * (of >> 1) + 1024 * c +
           16 * lane + 8 * (of & 1);
  }

  // The unit of a round: weights to LDS, their sums to l and r, m to the references that they
  // were taken against.
  struct Rows {
    u32x2 bytes;   // scales of the row
    u32x4 key[9];  // its pieces 4 s + group, as the first product takes them
  };
  __device__ __forceinline__ Rows rows(int round) const {
    Rows x;
    const uint32_t at = buffer(round);
    x.bytes = lds_read<u32x2>(at + kScalesAt + kScaleBytes * (kUnit * of + row));
    const uint32_t k_at = at + kUnitBytes * of + kNativeDataBytes * row + 16 * (group ^ turn(row));
#pragma unroll
    for (int s = 0; s < 9; ++s) x.key[s] = lds_read<u32x4>(k_at + 64 * s);
    return x;
  }
  // Bits of the unit's rows with an infinity or NaN.
  __device__ __forceinline__ uint32_t odd_rows(int round, const u32x2& bytes) const {
    // row `row`, pieces 9 group .. + 8
    const uint32_t mine = buffer(round) + kUnitBytes * of + kNativeDataBytes * row + 144 * group;
    uint32_t bad = 0;
#pragma unroll
    for (int n = 0; n < 9; ++n) {
      const u32x4 v = lds_read<u32x4>(mine + 16 * n);
      // (pieces 28 and up are the tail)
      const bool tail = 9 * group + n >= 28;
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= special(v[k], tail);
      if (n % 3 == 2) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int g = 0; g < 7; ++g) bad |= ((bytes[g / 4] >> (8 * (g % 4))) & 0xffu) == 0xffu;
    const uint64_t found = __ballot(bad != 0);
    return (uint32_t)(found | found >> 16 | found >> 32 | found >> 48) & 0xffffu;
  }
  template <bool kWhole>
  __device__ __forceinline__ void score(const Unit& x, int round, const Rows& in) {
    const u32x2 bytes = in.bytes;
    // rows of the unit that count
    const int stop = min(x.past ? past - x.at : held + a->nodes - x.at, kUnit);
    {  // shifts of row `row` for groups 2 group and 2 group + 1
      const uint32_t two = (group >= 2 ? bytes[1] : bytes[0]) >> (16 * (group & 1));
      const uint32_t to = lds + kShiftsAt + (round & 1) * kShiftsBytes + 512 * (of >> 1) +
                          128 * group + 16 * (row >> 2) + 2 * (4 * (of & 1) + (row & 3));
      const uint32_t both = (0x00fe00feu - ((two & 0xffu) | (two << 8 & 0xff0000u))) << 7;
      lds_write<uint16_t>(to, (uint16_t)both);
      lds_write<uint16_t>(to + 64, (uint16_t)(both >> 16));
    }
    f32x4 acc[2] = {};
#pragma unroll
    for (int s = 0; s < 7; ++s) {
      const float f = u2f(((bytes[s / 4] >> (8 * (s % 4))) & 0xffu) << 23);
      const u32x4 v = in.key[s];
      const bf16x8 k0 = codes8(v[0], v[1], f), k1 = codes8(v[2], v[3], f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, as_bf16x8(q[c][2 * s]), acc[c], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
        acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, as_bf16x8(q[c][2 * s + 1]), acc[c], 0, 0,
                                                         0);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bf16x8 k = as_bf16x8(in.key[7 + t]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, as_bf16x8(q[c][14 + t]), acc[c], 0, 0, 0);
    }
    // value i is row 4 group + i of the unit
    if (kWhole) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
        least = lower(lower(lower(least, acc[c][0]), acc[c][1]),
                      lower(acc[c][2], acc[c][3]));
    }
    uint32_t odd = 0, gone = 0;  // rows with an infinity or NaN, and with those nobody sees
    if (!kWhole) {
      // (a row with an infinity or NaN has a score like it with any query row: without one
      // no row is looked through)
      float none = 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) none = __builtin_fmaf(acc[c][i], 0.0f, none);
      if (__ballot(none != 0.0f) != 0) odd = odd_rows(round, bytes);
      gone = x.mapped ? odd | (0xffffu << stop & 0xffffu) : 0xffffu;
    }
    float top[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (!kWhole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 4 * group + i, p = x.at + n, node = p - held;
          const uint32_t word = node < 32 ? path[c][0] : path[c][1];
          const bool on_path = ((word >> (node & 31)) & 1u) != 0;
          const bool see = live[c] & x.mapped & (n < stop) &
                           (x.past | (node < 0 ? p >= lowest[c] : on_path));
          acc[c][i] *= a->scale_log2;
          acc[c][i] = (odd >> n) & 1u ? NAN : acc[c][i];
          acc[c][i] = see ? acc[c][i] : -INFINITY;
        }
      }
      // (a NaN, whose row leaves this query row NaN, moves no reference)
      top[c] = over_groups(
          higher(higher(acc[c][0], acc[c][1]), higher(acc[c][2], acc[c][3])), true);
      if (kWhole) top[c] *= a->scale_log2;
    }
    uint32_t moved = 0;
    if (__ballot((top[0] > m[0]) | (top[1] > m[1])) != 0) {
      moved = kMoved;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        advance(c, top[c] > m[c] ? ceilf(top[c]) + kHeadroom : m[c]);
        if (group == 0) lds_write(ref_at(round, of, c), m[c]);
      }
    }
    if (lane == 0) lds_write(lds + kStateAt + 16 * (round & 1) + 4 * of, gone | moved);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float ref = m[c] == -INFINITY ? 0.0f : m[c];
      f32x4 p;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = __builtin_amdgcn_exp2f(
            kWhole ? __builtin_fmaf(acc[c][i], a->scale_log2, -ref) : acc[c][i] - ref);
      l[c] += (p[0] + p[1]) + (p[2] + p[3]);
      p *= 0x1p127f;  // (in the exponent of exp2 it would cost the argument three bits)
      const bf16x2 lo = bf16_pair(p[0], p[1]), hi = bf16_pair(p[2], p[3]), one = {(__bf16)kUnit27,
                                                                                  (__bf16)kUnit27};
      r[c] = __builtin_amdgcn_fdot2_f32_bf16(lo, one, r[c], false);
      r[c] = __builtin_amdgcn_fdot2_f32_bf16(hi, one, r[c], false);
      const u32x2 d = {__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
      lds_write(weights_at(round, c), d);
    }
  }
  // Whether a row of the piece's whole units has an infinity. (Their NaN make scores and sums
  // NaN; an infinity whose score is -inf would weigh nothing.)
  __device__ __forceinline__ bool infinite_rows() const {
    bool found = false;
#pragma clang loop unroll(disable)
    for (int i = begin + of; i < end; i += kUnits) {
      const Unit x = unit(i, page_of(i));
      if (!whole(x)) continue;
      // row `row`, a quarter of its tail
      const u32x4* const from = (const u32x4*)(x.page + (x.in_page + row) * kNativeDataBytes +
                                               kNopeDim + 32 * group);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const u32x4 v = from[n];
#pragma unroll
        for (int k = 0; k < 4; ++k) found = found || special(v[k], true) != 0;
      }
    }
    return __ballot(found) != 0;
  }
  // The sums go on against `to`. (Equal references may both be infinite.)
  __device__ __forceinline__ void advance(int c, float to) {
    const float f = m[c] == to ? 1.0f : __builtin_amdgcn_exp2f(m[c] - to);
    l[c] *= f;
    r[c] *= f;
    m[c] = to;
  }
  // The highest reference of a round's units. (Those that did not move have the one that all
  // had before.)
  __device__ __forceinline__ void agree(int round, const u32x4& was) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float top = m[c];
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (uniform((int)(was[u] & kMoved))) top = fmaxf(top, lds_read<float>(ref_at(round, u, c)));
      advance(c, top);
    }
  }
  __device__ __forceinline__ static bool any_moved(const u32x4& was) {
    return (uniform((int)(was[0] | was[1] | was[2] | was[3])) & (int)kMoved) != 0;
  }

  __device__ __forceinline__ void run(int first_row) {
#pragma unroll
    for (int c = 0; c < 2; ++c) m[c] = -INFINITY, l[c] = r[c] = 0.0f;
    least = 0.0f;
    int parent = -2;
    if (lane < a->nodes) parent = a->parents[(int64_t)b * a->nodes + lane];
    int page = 0;
    if (begin + of < end) page = page_of(begin + of);
    asm volatile("" : "+v"(parent));  // (to be waited for before there are copies)
    copy_q(first_row);
    tree(first_row, parent);
    wait_copies<0>();
    lds_barrier();  // round 0's rows, and Q
    load_q();
    int round = 0;
#pragma clang loop unroll(disable)
    for (int from = begin; from < end; from += kUnits, ++round) {
      const int i = uniform(from + of);
      again();
      const u32x4 was = state(round - 1);
      const Rows in = rows(round);
      if (round > 0 && any_moved(was)) agree(round - 1, was);
      const Unit x = unit(min(i, units - 1), page);
      if (i + kUnits < end) page = page_of(i + kUnits);
      if (i < end) {
        if (whole(x))
          score<true>(x, round, in);
        else
          score<false>(x, round, in);
      } else {  // the round's last units: nothing
#pragma unroll
        for (int c = 0; c < 2; ++c) lds_write(weights_at(round, c), u32x2{0, 0});
        if (lane == 0) lds_write(lds + kStateAt + 16 * (round & 1) + 4 * of, 0xffffu);
      }
      lds_barrier();
    }
    if (round > 0) {
      const u32x4 was = state(round - 1);
      if (any_moved(was)) agree(round - 1, was);
    }
    // Only with a score of -inf (or NaN, which hides others) are the rows looked through: four
    // minima a round, which cost nothing, and no branch in it (16 x 16 nodes 117.8 us; 122 with one).
    if (__ballot(!(least > -INFINITY)) != 0 && infinite_rows()) l[0] = l[1] = NAN;
    // the row's sums; none of a row that sees nothing
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l[c] = over_groups(l[c], false);
      r[c] = over_groups(r[c], false);
      if (group == 0)
        lds_write(lds + kSumsAt + 8 * (kRows * of + 16 * c + row),
                  live[c] ? f32x2{l[c], r[c] * 0x1p-27f} : f32x2{0.0f, 0.0f});
    }
    lds_barrier();
  }
};

// Coordinates 128 g .. + 127 of all query rows: two groups of 64.
struct Adder : Tree {
  const int g;  // and unit g's copies
  uint32_t from[kCopies - 1];  // where the lane's piece of copy n is in the unit, less 1,024 n
  float m[2], sink[2];
  f32x4 o[2][2][4];  // query rows 16 c + row, coordinates 128 g + 64 h + 16 u + 4 group + i

  __device__ __forceinline__ Adder(const Tree& t) : Tree(t), g(wave - kScorers) {
#pragma unroll
    for (int n = 0; n < kCopies - 1; ++n) {
      const uint32_t p = 64 * n + lane, r = p / 36, j = p - 36 * r;
      from[n] = 576 * r + 16 * (j ^ turn(r)) - 1024 * n;
    }
  }

  // The rows of unit i, if there is one.
  __device__ __forceinline__ void copy(int i, int page, int round) const {
    if (i >= end) return;
    const uint32_t to = buffer(round) + kUnitBytes * g;
    const Unit x = unit(i, page);
    const uint8_t* const rows = x.page + x.in_page * kNativeDataBytes;
    copy_ahead16x4(rows, from[0], from[1], from[2], from[3], to);
    copy_ahead16x4(rows + 4096, from[4], from[5], from[6], from[7], to + 4096);
    copy_ahead16(rows + 8192, from[8], to + 8192);
    if (lane < kUnit * kScaleBytes / 4)
      copy_ahead4(x.page + kPageRecords * kNativeDataBytes + x.in_page * kScaleBytes, 4 * lane,
                  buffer(round) + kScalesAt + kUnit * kScaleBytes * g);
  }

  // Eight codes of the lane's coordinate of tile u of group k: of units 2 v and 2 v + 1, rows
  // 4 group .. + 3 each, as the second product's first operand takes them.
  __device__ __forceinline__ u32x2 codes(uint32_t at, int v, int k, int u) const {
    const int pair = row >> 1;  // the lane reads row 4 group + pair % 4 of unit pair / 4
    const int r = 4 * group + (pair & 3);
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(lds_void*)(uintptr_t)(
                   at + kUnitBytes * (pair >> 2) + kNativeDataBytes * r + 128 * g +
                   8 * (row & 1) + 16 * (u ^ turn(r)) + 64 * k + 2 * kUnitBytes * v)));
  }
  // The same of the tail, which is BF16.
  __device__ __forceinline__ u32x4 tail(uint32_t at, int v, int u) const {
    const int r = 4 * group + (row >> 2);
    u32x2 half[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)  // pieces 28 + 2 u and + 1
      half[k] = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)(uintptr_t)(
                     at + kNativeDataBytes * r + kNopeDim + 8 * (row & 1) +
                     kUnitBytes * (2 * v + k) + 64 * (u >> 1) +
                     16 * ((2 * (u & 1) + ((row & 3) >> 1)) ^ turn(r)))));
    return u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
  }
  // (asked again each time: kept, the answer takes a register too many)
  __device__ __forceinline__ bool with_tail() const {
    int mine = g;
    asm volatile("" : "+s"(mine));
    return mine == kAdders - 1;
  }

  // O += a round, in one stretch for all rounds, with everything asked for from LDS at once and
  // `between` while it comes. A round whose units took references of their own, or that leaves
  // rows out, only sets its operands right first.
  template <class F>
  __device__ __forceinline__ void add(int round, F between) {
    const uint32_t at = buffer(round);
    const u32x4 was = state(round);
    const uint32_t weights = lds + kWeightsAt + (round & 1) * kWeightsBytes + 16 * lane;
    const uint32_t shifts = lds + kShiftsAt + (round & 1) * kShiftsBytes + 128 * g + 16 * group;
    u32x4 p[2][2], shift[2][2], last[2][4];
    u32x2 first[2][4], second[2][4];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
#pragma unroll
      for (int c = 0; c < 2; ++c) p[v][c] = lds_read<u32x4>(weights + 2048 * v + 1024 * c);
      shift[0][v] = lds_read<u32x4>(shifts + 512 * v);
#pragma unroll
      for (int u = 0; u < 4; ++u) first[v][u] = codes(at, v, 0, u);
    }
    if (!with_tail()) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        shift[1][v] = lds_read<u32x4>(shifts + 512 * v + 64);
#pragma unroll
        for (int u = 0; u < 4; ++u) second[v][u] = codes(at, v, 1, u);
      }
    } else {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        shift[1][v] = u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};  // 127 << 7
#pragma unroll
        for (int u = 0; u < 4; ++u) last[v][u] = tail(at, v, u);
      }
    }
    const uint32_t any = (uint32_t)uniform((int)(was[0] | was[1] | was[2] | was[3]));
    if (any & kMoved) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float own[kUnits], top = m[c];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const float ref = lds_read<float>(ref_at(round, u, c));
          own[u] = was[u] & kMoved ? ref : m[c];
          top = fmaxf(top, own[u]);
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          // whole log2 units down, in both exponents; 255: past every exponent, also for a
          // difference that is NaN (infinities: the row's sum is NaN then)
          const uint32_t d = __umul24((uint32_t)fminf(top - own[u], 255.0f), 0x00800080u);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            p[u / 2][c][2 * (u % 2) + k] = sub_sat(p[u / 2][c][2 * (u % 2) + k], d);
        }
        const float f = m[c] == top ? 1.0f : __builtin_amdgcn_exp2f(m[c] - top);
        m[c] = top;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int u = 0; u < 4; ++u) o[c][k][u] *= f;
      }
    }
    if (any & (kMoved - 1)) {
#pragma unroll
      for (int n = 0; n < kUnits; ++n) {  // rows 4 group .. + 3 of unit n
        const uint32_t four = was[n] >> (4 * group);
        const uint32_t lo = (four & 1u ? 0u : 0xffffu) | (four & 2u ? 0u : 0xffff0000u);
        const uint32_t hi = (four & 4u ? 0u : 0xffffu) | (four & 8u ? 0u : 0xffff0000u);
        const uint32_t bytes = (lo & 0xffu) | (lo >> 8 & 0xff00u) | (hi << 16 & 0xff0000u) |
                               (hi & 0xff000000u);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          first[n / 2][u][n % 2] &= bytes;
          if (!with_tail()) {
            second[n / 2][u][n % 2] &= bytes;
          } else {
            last[n / 2][u][2 * (n % 2)] &= lo;
            last[n / 2][u][2 * (n % 2) + 1] &= hi;
          }
        }
      }
    }
    between();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && !with_tail()) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            last[v][u] =
                __builtin_bit_cast(u32x4, codes8(second[v][u][0], second[v][u][1], 1.0f));
      }
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        bf16x8 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          x[u] = k == 0 ? codes8(first[v][u][0], first[v][u][1], 1.0f) : as_bf16x8(last[v][u]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = sub_sat(p[v][c][i], shift[k][v][i]);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            o[c][k][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[u], as_bf16x8(w), o[c][k][u],
                                                                 0, 0, 0);
        }
      }
    }
  }

  __device__ __forceinline__ void run(int first_row) {
    const int i = uniform(begin + g);
    int page = 0;
    if (i < end) page = page_of(i);
    copy(i, page, 0);
    if (i + kUnits < end) page = page_of(i + kUnits);
    copy(i + kUnits, page, 1);
    if (i + 2 * kUnits < end) page = page_of(i + 2 * kUnits);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[c] = -INFINITY;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[c][k][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // (for the end, so that it need not wait for them: 7 trees of 5 nodes 13.0 us, 12.6 so)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sink[c] = -INFINITY;
      const int at = first_row + 16 * c + row;
      if (a->sink && of_slots == 1 && at < a->q_rows) sink[c] = a->sink[at % a->heads];
    }
    landed(i + kUnits);  // round 0 (and what was asked for besides counts as round 1's)
    lds_barrier();
    // scored: round; added: the one before; copied: the one after next
    if (begin < end) {
      const int i = uniform(begin + g) + 2 * kUnits;
      copy(i, page, 2);
      if (i + kUnits < end) page = page_of(i + kUnits);
      landed(i);
    }
    lds_barrier();
    int round = 1;
#pragma clang loop unroll(disable)
    for (int from = begin; from < end; from += kUnits, ++round) {
      const int i = uniform(from + g) + 3 * kUnits;
      add(round - 1, [&] { copy(i, page, round + 2); });
      if (i + kUnits < end) page = page_of(i + kUnits);
      landed(i);
      lds_barrier();
    }
    anew();
    finish(first_row);
  }

  // Until the copies before those of unit `last`, the latest, have landed.
  __device__ __forceinline__ void landed(int last) const {
    if (last < end)
      wait_copies<kCopies>();
    else
      wait_copies<0>();
  }

  __device__ __forceinline__ void finish(int first_row) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = 0.0f, rsum = 0.0f;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const f32x2 part = lds_read<f32x2>(lds + kSumsAt + 8 * (kRows * u + 16 * c + row));
        sum += part[0];
        rsum += part[1];
      }
      const int at = first_row + 16 * c + row;
      if (at >= a->q_rows) continue;
      const int node = at / a->heads, h = at - node * a->heads;
      const int64_t token = (int64_t)b * a->nodes + node;
      const int c0 = 128 * g + 4 * group;
      if (of_slots > 1) {
        const int64_t to = (token * a->slots + slot) * a->heads + h;
        const float f = sum != 0.0f ? 1.0f / rsum : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          f32x4 x = o[c][u / 4][u % 4] * f;
          if (sum == 0.0f) x = f32x4{0.f, 0.f, 0.f, 0.f};
          __builtin_nontemporal_store(x, (f32x4*)(a->ws_o + to * kHeadDim + c0 + 16 * u));
        }
        // (NaN goes on as infinity: the combine's maximum would pass over a NaN)
        if (g == 0 && group == 0)
          a->ws_lse[to] = sum != sum     ? INFINITY
                         : sum != 0.0f ? m[c] + __builtin_amdgcn_logf(sum)
                                       : -INFINITY;
        continue;
      }
      const float sink2 = sink[c] * kLog2e;
      const float top = fmaxf(sum != 0.0f ? m[c] : -INFINITY, sink2);
      float f = 0.0f, lse = -INFINITY;
      if (top != -INFINITY || sum != 0.0f) {
        const float em = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[c] - top);
        const float z = sum * em + __builtin_amdgcn_exp2f(sink2 - top);
        // (O over the rounded weights' sum, times the rows' share of Z)
        if (sum != 0.0f) f = sum * em / (rsum * z);
        lse = (top + __builtin_amdgcn_logf(z)) * kLn2;
      }
      if (g == 0 && group == 0) a->lse[token * a->heads + h] = lse;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        f32x4 x = o[c][u / 4][u % 4] * f;
        if (sum == 0.0f) x = f32x4{0.f, 0.f, 0.f, 0.f};
        *(u32x2*)(a->out + (token * a->heads + h) * kHeadDim + c0 + 16 * u) =
            u32x2{__builtin_bit_cast(uint32_t, bf16_pair(x[0], x[1])),
                  __builtin_bit_cast(uint32_t, bf16_pair(x[2], x[3]))};
      }
    }
  }
};

// The rounds of all requests stand on one axis, each request's followed by kOverhead, and a
// part takes an equal piece of it: b's rounds from `start` on, of which several parts can have
// some. Starts go to LDS.
struct Share {
  int first;  // request
  int begin, end, size;
};
__device__ __forceinline__ Share deal(const Tree& t, int part) {
  const_args* const a = t.a;
  int total = 0, most = 0;
  for (int i0 = 0; i0 < a->batch; i0 += 64) {
    const int i = i0 + t.lane;
    int cost = 0;
    if (i < a->batch)
      cost = kOverhead + Tree::rounds(Tree::extent(
                             a, a->lengths[i], a->past_lengths ? a->past_lengths[i] : 0));
    const int upto = (int)wave_prefix((uint32_t)cost);
    // (each wave writes all of them: it waits for nobody)
    if (i <= a->batch) lds_write(t.lds + kStartsAt + 4 * i, total + upto - cost);
    total += __builtin_amdgcn_readlane(upto, 63);
    most = max(most, cost - kOverhead);
  }
  if (a->batch % 64 == 0) lds_write(t.lds + kStartsAt + 4 * a->batch, total);
  most = uniform((int)wave_all<true>((float)most));
  Share x;
  // (and no request in more pieces than there are slots; one can begin inside a part, but for
  // the first)
  const int cuts = max(a->slots - (a->batch > 1 ? 1 : 0), 1);
  x.size = max(max((total - kOverhead + a->parts - 1) / a->parts, (most + cuts - 1) / cuts), 1);
  x.begin = part * x.size;
  x.end = x.begin + x.size;
  x.first = 0;
  for (int i0 = 0; i0 < a->batch; i0 += 64) {
    const int i = i0 + t.lane;
    const int next = lds_read<int>(t.lds + kStartsAt + 4 * min(i + 1, a->batch));
    x.first += __popcll(__ballot(i < a->batch && next - kOverhead <= x.begin));
  }
  return x;
}

__global__ __launch_bounds__(64 * (kScorers + kAdders)) void tree_decode_kernel(TreeArgs) {
  const_args* a = (const_args*)__builtin_amdgcn_kernarg_segment_ptr();
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLdsBytes];
  // Workgroups go to the eight XCDs in turn: the tiles of one part, which read the same rows,
  // go to one, so that its L2 cache serves all but the first. An XCD takes every eighth part if
  // that fills none with more than its 32 CUs hold, or if there are many requests, which may
  // come in the order of their lengths; otherwise parts that follow each other, all XCDs as
  // many tiles (5 requests x 62 tiles: 27 us so, 50 with every eighth).
  const int xcd = (int)blockIdx.x & 7, turn = (int)blockIdx.x >> 3;
  const int at = a->each_eighth ? (turn / a->tiles * 8 + xcd) * a->tiles + turn % a->tiles
                                : xcd * ((int)gridDim.x >> 3) + turn;
  const int part = at / a->tiles;
  const int tile = at - part * a->tiles, first_row = tile * kRows;
  Tree t(a, (uint32_t)(uintptr_t)(lds_void*)lds);
  if (part >= (a->parts > 0 ? a->parts : a->batch)) return;
  Share share = {part, 0, 0, 0};
  if (a->parts > 0) share = deal(t, part);
  const int last = a->parts > 0 ? a->batch : part + 1;
  const auto start = [&](int i) { return uniform(lds_read<int>(t.lds + kStartsAt + 4 * i)); };
  const auto each = [&](auto run) {
#pragma clang loop unroll(disable)
    for (int b = uniform(share.first); b < last; ++b) {
      int from = 0, to = 0x7fffffff / kUnits;
      t.slot = 0, t.of_slots = 1;
      if (a->parts > 0) {
        const int at = start(b), rounds = start(b + 1) - kOverhead - at;
        int size = share.size;  // (nor is its reciprocal kept)
        asm volatile("" : "+s"(size));
        if (at >= share.end) break;
        from = max(share.begin - at, 0), to = min(share.end - at, rounds);
        t.slot = part - at / size;
        t.of_slots = (at + rounds - 1) / size - at / size + 1;
        if (a->counts && tile == 0 && t.slot == t.of_slots - 1 && threadIdx.x == 0)
          a->counts[b] = t.of_slots > 1 ? t.of_slots : 0;
      }
      t.piece(b, from, to);
      int row = first_row;
      asm volatile("" : "+s"(row));
      run(row);
    }
  };
  if (t.wave < kScorers)
    each([&](int row) { Scorer(t).run(row); });
  else
    each([&](int row) { Adder(t).run(row); });
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

bool bad_sizes(int64_t batch, int64_t nodes, int64_t heads, int64_t blocks, int64_t window,
               int64_t past_blocks) {
  return batch < 0 || nodes < 0 || nodes > kMaxNodes || heads < 0 || heads > kMaxHeads ||
         batch > 65535 || batch * nodes > 65535 || blocks < 0 || blocks > (1 << 24) ||
         window < 0 || window > 0x7fffffff || past_blocks < 0 || past_blocks > (1 << 24);
}

struct Plan {
  int parts, slots;
  size_t counts_at, bytes;
};
// Parts: as many as fill the chip with one turn of workgroups (one a CU, for its LDS), four
// turns where a turn could not be filled well. With four turns of whole requests or more, a
// request each, as in any order they fill it; and with requests of few rounds, as a piece and
// the combine cost what 6 rounds take.
constexpr int64_t kWhole = 6;
Plan plan(int64_t batch, int64_t nodes, int64_t heads, int64_t blocks, int64_t window,
          int64_t past_blocks) {
  const int64_t tiles = std::max<int64_t>((nodes * heads + kRows - 1) / kRows, 1);
  int64_t rows = blocks * kPageRecords;
  if (window > 0) rows = std::min(rows, window + nodes + kUnit);
  const int64_t rounds =
      std::max<int64_t>((rows + past_blocks * kPageRecords + kRound - 1) / kRound, 1);
  Plan p = {0, 1, 0, 0};
  if (batch > kMaxShared || batch * tiles >= 1024 || rounds <= kWhole || rounds >= (1 << 22))
    return p;
  const int64_t most = std::max<int64_t>(batch * rounds, 1);
  p.parts = (int)std::min<int64_t>(std::max<int64_t>((tiles <= 64 ? 256 : 1024) / tiles, 1), most);
  if (batch <= 1) {
    const int64_t share = (rounds + p.parts - 1) / p.parts;
    p.slots = (int)((rounds + share - 1) / share);
  } else {  // four times an even share's
    p.slots = (int)std::min<int64_t>(4 * ((p.parts + batch - 1) / batch) + 1, p.parts);
  }
  p.slots = std::min(p.slots, kMaxSplits);
  if (p.slots > 1) {
    p.counts_at = (size_t)(p.slots * batch * nodes * heads) * (kHeadDim + 1) * sizeof(float);
    p.bytes = p.counts_at + (size_t)batch * sizeof(int32_t);
  }
  return p;
}

}  // namespace

extern "C" int rm_tree_decode_workspace(int64_t batch, int64_t nodes, int64_t heads,
                                        int64_t max_blocks, int64_t window, int64_t history_blocks,
                                        int32_t* num_splits, size_t* workspace_bytes) {
  if (bad_sizes(batch, nodes, heads, max_blocks, window, history_blocks)) return RM_ERR_SHAPE;
  const Plan p = plan(batch, nodes, heads, max_blocks, window, history_blocks);
  if (num_splits) *num_splits = p.slots;
  if (workspace_bytes) *workspace_bytes = p.bytes;
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
  const Plan p = plan(batch, nodes, heads, max_blocks, window, history_blocks);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return RM_ERR_WORKSPACE;
  if (p.bytes > 0 && !aligned(workspace, 16)) return RM_ERR_ALIGN;
  TreeArgs a;
  a.q = q;
  a.batch = (int)batch;
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
  a.scale_log2 = std::fabs(softmax_scale) * kLog2e;
  a.negated = softmax_scale < 0.0f;
  a.parts = p.parts;
  a.each_eighth = p.parts > 0 ? (p.parts + 7) / 8 * a.tiles <= 32 : batch >= 64;
  a.slots = p.slots;
  a.out = out;
  a.lse = lse;
  a.ws_o = p.slots > 1 ? (float*)workspace : nullptr;
  a.ws_lse = p.slots > 1 ? a.ws_o + (size_t)p.slots * rows * kHeadDim : nullptr;
  a.counts = p.slots > 1 ? (int32_t*)((uint8_t*)workspace + p.counts_at) : nullptr;
  const int64_t parts = p.parts > 0 ? p.parts : batch;
  const int64_t groups = a.each_eighth ? (parts + 7) / 8 * 8 * a.tiles
                                       : (parts * a.tiles + 7) / 8 * 8;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(tree_decode_kernel, dim3((unsigned)groups),
                     dim3(64 * (kScorers + kAdders)), 0, s, a);
  if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  if (p.slots > 1) {
    launch_combine<true, true>(a.ws_o, a.ws_lse, sink, p.slots, batch * nodes, heads, out, lse, s,
                               a.counts, batch);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  return RM_OK;
}
