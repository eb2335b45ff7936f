// Sparse-MLA decode over 4-bit records, jointly with sliding-window rows of a
// Native pool. For query token t and head h, over the valid entries j of t's list
// and window (K_j the dequantized 512-coordinate row, V = K):
//   l_j = (q_h . K_j) * scale, Z = sum_j exp(l_j) + exp(sink_h),
//   out = sum_j exp(l_j) K_j / Z, lse = ln Z.
//
// A workgroup owns (split, token, 16 heads) and takes its share of the list in rounds of
// kWaves / 2 chunks of 32 records (chunks are dealt to the splits and then in turn), then
// its share of the window, 16 rows a wave and round. kWaves waves compute, half as many
// more copy; one barrier a round. In the time between two barriers
//   * a computing wave scores 16 records of round i: S^T = K Q^T on
//     v_mfma_f32_16x16x32_bf16, Q in registers; it leaves in LDS the weights P = 2^(s -
//     m) as BF16, m the running maximum (in whole log2 units) as far as the wave knows
//     it, or where a score passes that by 2^24, the unit above the tile's largest (weights
//     of up to 2^24 are no loss in a floating format), and the records' scale exponents;
//   * and adds all of round i - 1 to the 512 / kWaves output coordinates it owns: O^T +=
//     V^T P^T. The codes come out of LDS transposed (ds_read_b64_tr_b4) and become BF16
//     without their scales: those are powers of two that differ by record and group, so
//     they go to the weights, and so does, where the round has any, the step from a
//     tile's m to the running maximum: integer subtractions on the BF16 exponents, two
//     weights an instruction, saturating at zero (v_pk_sub_u16 clamp), against the largest
//     scale the store writes, 2^32; O is in units of it. A weight that a scale takes below
//     2^-126 becomes zero: less than 2^-78 of the largest weight (in (1/2, 2^24]) even at the
//     smallest scale the store writes, 2^-15. A record with a scale past 2^32 is made NaN.
//     The output is divided by the sum of the weights as they were rounded, and lse takes
//     the sum of the exact ones: roundings that a token's weights have in common cancel
//     (one entry gives its record exactly). Against the definition in 64 bits, relative to
//     an output rounded once: 1.5 times that error for one entry without it and 1.0 with
//     it, 1.4 and 1.2 for 8 to 500, for 1 % of the time;
//   * the copying waves fetch round i + 2 into the LDS that round i - 2 has left
//     (global_load_lds, consecutive lanes taking consecutive 16-byte pieces of a record,
//     17 a record, so that a copy touches each 128-byte line once), and wait for round
//     i + 1. Waves that both computed and copied spent 40 % of a round held up at the
//     issue of copies, with the memory idle for the rest of it.
// P^T in LDS is what the lane holding it writes: the order of the records in the second
// product's long axis is free, and S^T's is taken.
//
// 256 tokens x 2,048 records at random places: 45 us (143 MB of records, 3.2 TB/s; a kernel
// that does nothing but gather them takes 32 to 34). About 8 us are the start; the rest is
// bound by that gather, with the vector pipes issuing in 50 % of the cycles (23.5
// instructions a record, a third of them the two conversions of its codes) and the matrix
// pipes busy in 17 %. 64 tokens x 2,048: 19.3 us and 4.1 the combine, 1 token 7.1 and 3.0
// (traced).
// Before the copying waves had their own turn: 58; with one accumulator of all coordinates
// a wave, merged at the end: 57.9; with records prefetched into registers: 77.
//
// At the start the list's entries, the block-table row (into LDS, up to kTableCache
// columns), the lengths and Q are all requested together, so that the first records wait
// for two round trips of memory and not for four.
#include <algorithm>

#include "combine.h"
#include "mx4_device.h"
#include "remnant_mi355x.h"

using namespace rm;

namespace {

constexpr int kMaxTopk = 1 << 20;
constexpr int kMaxWindow = 512;
constexpr int kMaxHeads = 1024;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

struct DecodeArgs {
  int first;  // token of workgroups (., 0, .)
  const uint16_t* q;
  uint64_t q_len_magic;  // ceil(2^32 / q_len): token t < 2^16 is of request t * q_len_magic >> 32
  int heads;
  const uint8_t* pool;
  int pool_pages;
  bool once;  // the list's records are read with copy16_once()
  const int32_t* block_table;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* seqlens;
  const int32_t* indices;
  int topk;
  const int32_t* topk_length;
  const uint8_t* swa_pool;
  int64_t swa_rows;
  const int32_t* swa_indices;
  int swa_topk;
  const int32_t* swa_length;
  const float* sink;
  float scale_log2;
  int splits;        // workgroups (along x) that share a token's list
  int window_split;  // the one that takes the window: one more, or 0 where there is one only
  uint64_t splits_magic;  // ceil(2^32 / splits): x / splits = x * splits_magic >> 32 for x < 2^17
  int ws_splits;  // partial slots a row; 0: finish in place
  uint16_t* out;
  float* lse;
  float* ws_o;    // [this launch's tokens, ws_splits, heads, 512]
  float* ws_lse;  // [the same, ws_splits, heads]
};

// A chunk in LDS: its records 272 bytes apart (4 banks), with 128 bytes between the
// first 16 (tile 0) and the second, so that the transposed reads of a lane group's 2 x 4
// records meet no bank twice. 552 pieces of 16 bytes, 9 copies.
constexpr int kTilePieces = 16 * 17 + 8;
constexpr int kTileBytes = 16 * kTilePieces;                     // 4,480
constexpr int kChunkBytes = kTileBytes + 16 * kMx4RecordBytes;   // 8,832
constexpr int kCopies = 9;
constexpr int kLastLanes = 2 * kTilePieces - 8 - 64 * (kCopies - 1);  // of the last copy: 40
constexpr int kBuffers = 4;  // rounds in LDS: being added, being scored, two being copied
constexpr int kBatch = 16;   // rounds whose slots are looked up together
constexpr int kTableCache = 1024;  // block-table columns kept in LDS
// A window chunk: 16 rows, 16-byte piece 4 j + g of row r at 1024 j + 256 g + 16 r, then
// the scale bytes by group.
constexpr int kWindowScalesAt = 16 * kNativeDataBytes;
constexpr int kWindowBytes = kWindowScalesAt + 128;
constexpr int kScaleRef = 127 + kMx4MaxExponent;
constexpr int kSmallPool = 246723;  // pages whose bytes have 32-bit numbers
static_assert((int64_t)kSmallPool * kPageRecords * kMx4RecordBytes <= 0xffffffff, "4 GiB");
constexpr int64_t kOnceBytes = 64 << 20;
constexpr float kSlack = 24.0f;  // log2 units a score may pass the running maximum by

// LDS of a workgroup: the rounds' chunks (or a window chunk a wave); then, twice (odd and
// even rounds), by chunk the weights (16 bytes a lane, tile 0's and tile 1's four; a
// window chunk: four floats) and the scale exponents [16 groups][32 record slots] u16, (159
// - scale byte) << 7, and by tile the references of the 16 heads; then the block-table row.
// Q passes through the middle at the start, a head's row every 1,040 bytes (4 banks).
template <int kWaves>
struct Lds {
  static constexpr int kChunks = kWaves / 2;
  static constexpr int kRound = kChunks * kChunkBytes;
  static constexpr int kWeights = kBuffers * kRound;
  static constexpr int kShifts = kWeights + 2 * kChunks * 1024;
  static constexpr int kTops = kShifts + 2 * kChunks * 1024;
  static constexpr int kEnd = kTops + 2 * kWaves * 64;
  static constexpr int kQPitch = 1040;
  static constexpr int kTable = kEnd > kWeights + 16 * kQPitch ? kEnd : kWeights + 16 * kQPitch;
  static constexpr int kLive = kTable + 4 * kTableCache;  // [kBuffers][kChunks] bit masks
  static constexpr int kMoved = kLive + 4 * kBuffers * kChunks;  // [4]: a round moves m
  static constexpr int kEarly = kMoved + 16;                     // [kWaves][16] window slots
  static constexpr int kBytes = kEarly + 64 * kWaves;
  static_assert(kBytes <= 160 * 1024 && kWaves * kWindowBytes <= kWeights, "LDS of a CU");
};

// Copies HBM -> LDS: 16 bytes a lane to lds + 16 lane. The LDS address is a plain number,
// so that the compiler ties the copies to no array; wait_copies() orders them.
__device__ __forceinline__ void copy16(const void* src, uint32_t lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)__builtin_amdgcn_readfirstlane(lds),
                                   16, 0, 0);
}
// The same, of data that the caches will not see again: calls whose lists hold kOnceBytes
// of records or more (256 tokens x 2,048 records, 143 MB, 48.4 -> 46.4 us; 64 tokens, 36 MB,
// which three calls in turn find in the last-level cache, 22.7 -> 23.4).
__device__ __forceinline__ void copy16_once(const void* src, uint32_t lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)__builtin_amdgcn_readfirstlane(lds),
                                   16, 0, 2);
}
__device__ __forceinline__ void copy4(const void* src, uint32_t lds) {
  __builtin_amdgcn_global_load_lds(src, (lds_void*)(uintptr_t)__builtin_amdgcn_readfirstlane(lds),
                                   4, 0, 0);
}
// Until at most kLater vector loads issued since are in flight.
template <int kLater>
__device__ __forceinline__ void wait_copies() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kLater & 15) | ((kLater >> 4) << 14));
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  __builtin_amdgcn_sched_barrier(0);
}
template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)at;
}
template <class T>
__device__ __forceinline__ void lds_write(uint32_t at, T v) {
  *(__attribute__((address_space(3))) T*)(uintptr_t)at = v;
}
// Over the four lanes that share lane % 16.
__device__ __forceinline__ float over_groups_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = fmaxf(u2f(a[0]), u2f(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(b[0]), u2f(b[1]));
}
__device__ __forceinline__ float over_groups_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = u2f(a[0]) + u2f(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return u2f(b[0]) + u2f(b[1]);
}
// Barrier that orders LDS accesses only: loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
__device__ __forceinline__ uint32_t sub_sat(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, a),
                                                          __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// What the waves of a workgroup share.
template <int kWaves>
struct Share {
  const DecodeArgs& a;
  const uint32_t lds;
  const int lane, wave, split;
  const int64_t t;
  int live, rows, records;  // entries of the list and the window; records of the request
  int chunks, back;         // the split's chunks of the list and the window
  int rounds;

  __device__ __forceinline__ Share(const DecodeArgs& args, uint32_t lds_at)
      : a(args),
        lds(lds_at),
        lane(wave_lane()),
        wave(uniform((int)(threadIdx.x >> 6))),
        split((int)blockIdx.x),
        t(args.first + (int)blockIdx.y) {}
  __device__ __forceinline__ int64_t request() const {
    return (int64_t)(((uint64_t)t * a.q_len_magic) >> 32);
  }
  __device__ __forceinline__ void lengths() {
    live = a.topk, rows = a.swa_topk, records = 0x7fffffff;
    if (a.topk_length) live = max(min(a.topk_length[t], live), 0);
    if (a.swa_length) rows = max(min(a.swa_length[t], rows), 0);
    if (a.seqlens) records = a.seqlens[request()];
    // list chunks split, split + splits, ...; the window in one workgroup
    chunks = split < a.splits ? (int)(((uint64_t)((live + 31) / 32 - split + a.splits - 1) *
                                       a.splits_magic) >> 32) : 0;
    back = split == a.window_split ? (rows + 15) / 16 : 0;
    rounds = (chunks + kWaves / 2 - 1) / (kWaves / 2);
  }
};

// A copying wave: chunk `wave - kWaves` of every round.
template <int kWaves>
struct Copier : Share<kWaves> {
  using L = Lds<kWaves>;
  using S = Share<kWaves>;
  using S::a, S::lds, S::lane, S::wave, S::split, S::t;
  const int of;  // the chunk of a round
  const int32_t *idx, *table;
  // Copy n takes piece 64 n + lane: of record from / 4 of the chunk, bytes off .. off + 15
  // (the 8 pieces between the tiles copy some piece again). from | off << 8
  uint32_t where[kCopies];
  int slots[kBatch / 2];  // lane: entry lane % 32 of round 2 e + lane / 32; -1: no record

  __device__ __forceinline__ Copier(const DecodeArgs& args, uint32_t lds_at)
      : S(args, lds_at), of(S::wave - kWaves) {
    idx = a.indices + t * a.topk;
    table = a.block_table + this->request() * a.bt_stride;
  }
  // Entry of the list that slots[0] of a batch stands for, and how far on slots[1]'s is.
  __device__ __forceinline__ int entry(int first) const {
    const int c = (first + (lane >> 5)) * L::kChunks + of;
    return 32 * (c * a.splits + split) + (lane & 31);
  }
  __device__ __forceinline__ int stride() const { return 64 * L::kChunks * a.splits; }
  // The first batch's entries, as far as the list's capacity goes: the length comes beside.
  __device__ __forceinline__ void ask() {
    const int k = entry(0);
#pragma unroll
    for (int e = 0; e < kBatch / 2; ++e) {
      slots[e] = -1;
      if (e * stride() < a.topk) slots[e] = idx[min(k + e * stride(), a.topk - 1)];
    }
#pragma unroll
    for (int n = 0; n < kCopies; ++n) {
      const int p = 64 * n + lane, tile = p >= kTilePieces;
      const int in_tile = min(p - tile * kTilePieces, 16 * 17 - 1);
      const int r = in_tile * 241 >> 12;  // / 17, for numbers below 272
      where[n] = (uint32_t)(4 * (16 * tile + r)) | (uint32_t)(16 * (in_tile - 17 * r)) << 8;
    }
  }
  // slots[kFrom] .. [kTo - 1]: from entries (the first batch's are there) to record numbers.
  template <int kFrom, int kTo>
  __device__ __forceinline__ void look_up(int first) {
    const bool cached = a.max_blocks <= kTableCache;
    const int k = entry(first);
    int page[kBatch / 2];
    if (first > 0) {
#pragma unroll
      for (int e = kFrom; e < kTo; ++e)
        slots[e] = k + e * stride() < this->live ? idx[k + e * stride()] : -1;
    }
#pragma unroll
    for (int e = kFrom; e < kTo; ++e) {
      const int r = k + e * stride() < this->live ? slots[e] : -1;
      const bool inside = r >= 0 && r < this->records && (r >> 6) < a.max_blocks;
      page[e] = -1;
      if (cached)
        page[e] = lds_read<int>(lds + L::kTable + 4 * (inside ? r >> 6 : 0));
      else if (inside)
        page[e] = table[r >> 6];
      if (!inside) page[e] = -1;
    }
#pragma unroll
    for (int e = kFrom; e < kTo; ++e)
      slots[e] = page[e] >= 0 && page[e] < a.pool_pages
                     ? page[e] * kPageRecords + (slots[e] & 63) : -1;
  }
  // The rest of the first batch, when rounds 0 and 1 have been copied and slots moved down.
  __device__ __forceinline__ void look_up_later() {
    int rest[kBatch / 2];
#pragma unroll
    for (int e = 0; e + 1 < kBatch / 2; ++e) rest[e + 1] = slots[e];
#pragma unroll
    for (int e = 1; e < kBatch / 2; ++e) slots[e] = rest[e];
    look_up<1, kBatch / 2>(0);
#pragma unroll
    for (int e = 1; e < kBatch / 2; ++e) slots[e - 1] = slots[e];
  }
  // Chunks that the last round does not have are neither copied nor added (1 token x 129
  // records 8.4 -> 7.7 us, 16 tokens x 64 heads x 317 13.4 -> 12.8).
  __device__ __forceinline__ bool has(int i) const { return i * L::kChunks + of < this->chunks; }
  // Until round i has landed, of which round i + 1's copies, if there are any, came later.
  __device__ __forceinline__ void landed(int i) const {
    if (has(i + 1))
      wait_copies<kCopies>();
    else
      wait_copies<0>();
  }
  // The chunk of round i; its live records go to LDS.
  __device__ __forceinline__ void copy(int i) {
    const int of_round = slots[0];
    if (i & 1) {  // (rounds come in turn)
#pragma unroll
      for (int e = 1; e < kBatch / 2; ++e) slots[e - 1] = slots[e];
    }
    const uint32_t to = lds + (i & (kBuffers - 1)) * L::kRound + of * kChunkBytes;
    const uint32_t live_at = lds + L::kLive + 4 * ((i & (kBuffers - 1)) * L::kChunks + of);
    const uint32_t mask = (uint32_t)(__ballot(of_round >= 0) >> (32 * (i & 1)));
    if (lane == 0) lds_write(live_at, mask);
    if (!has(i)) return;
    const int record = max(of_round, 0);
    const int base = 128 * (i & 1);
    const bool all = lane < kLastLanes;
    if (a.pool_pages <= kSmallPool) {  // 32-bit offsets from the pool
      const int at = (int)((uint32_t)record * kMx4RecordBytes);
      uint32_t off[kCopies];
#pragma unroll
      for (int n = 0; n < kCopies; ++n)
        off[n] = (uint32_t)__builtin_amdgcn_ds_bpermute(base + (int)(where[n] & 0xff), at);
#pragma unroll
      for (int n = 0; n < kCopies; ++n) off[n] += where[n] >> 8;
      if (a.once) {
#pragma unroll
        for (int n = 0; n < kCopies; ++n)
          if (n < kCopies - 1 || all) copy16_once(a.pool + off[n], to + 1024 * n);
      } else {
#pragma unroll
        for (int n = 0; n < kCopies; ++n)
          if (n < kCopies - 1 || all) copy16(a.pool + off[n], to + 1024 * n);
      }
    } else {
#pragma unroll
      for (int n = 0; n < kCopies; ++n) {
        const int slot = __builtin_amdgcn_ds_bpermute(base + (int)(where[n] & 0xff), record);
        if (n < kCopies - 1 || all)
          copy16_once(a.pool + ((int64_t)slot * kMx4RecordBytes + (where[n] >> 8)), to + 1024 * n);
      }
    }
  }
  __device__ __forceinline__ void run() {
    __builtin_amdgcn_s_setprio(3);
    ask();
    this->lengths();
    lds_barrier();  // the block-table row
    const int rounds = this->rounds;
    if (rounds > 0) {
      look_up<0, 1>(0);  // rounds 0 and 1; the others' while their records are on the way
      copy(0);
      if (rounds > 1) {
        copy(1);
        if (rounds > 2) look_up_later();
        landed(0);
      } else {
        wait_copies<0>();
      }
    }
    lds_barrier();
    for (int i = 0; i < rounds; ++i) {
      if (i + 2 < rounds) {
        if (((i + 2) & (kBatch - 1)) == 0) look_up<0, kBatch / 2>(i + 2);
        copy(i + 2);
        landed(i + 1);
      } else {
        wait_copies<0>();
      }
      lds_barrier();
    }
  }
};

// 2^(from - to) for running maxima, 1 where both are -inf (nothing yet).
__device__ __forceinline__ float step_down(float from, float to) {
  return from == to ? 1.0f : __builtin_amdgcn_exp2f(from - to);
}

// A computing wave.
template <int kWaves>
struct Decode : Share<kWaves> {
  using L = Lds<kWaves>;
  using S = Share<kWaves>;
  using S::a, S::lds, S::lane, S::wave, S::split, S::t;
  static constexpr int kTiles = kHeadDim / 16 / kWaves;  // 16-coordinate tiles of O a wave
  const int row, group;  // row: record of a tile, or head; group: lane / 16
  const int h0;
  bf16x8 q[16];     // q[4 j + u]: coordinates 128 j + 32 group + 8 u .. + 7 of head `row`
  f32x4 o[kTiles];  // coordinate 16 tile + 4 group + i of the wave's, of head `row`
  float m;          // running maximum of head `row` (whole log2 units)
  float l, r;       // this lane's sums of weights: as they are, and as rounded to BF16
  float owns;       // reference of the wave's last tile, sums of its weights against it
  float sums, rsums;

  __device__ __forceinline__ Decode(const DecodeArgs& args, uint32_t lds_at)
      : S(args, lds_at),
        row(S::lane & 15),
        group(S::lane >> 4),
        h0(blockIdx.z * 16),
        m(-INFINITY),
        l(0.0f),
        r(0.0f) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] = zero_f();
  }
  static __device__ __forceinline__ f32x4 zero_f() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

  // Q: the waves copy the 16 heads' rows to LDS ...
  __device__ __forceinline__ void copy_q() const {
#pragma unroll
    for (int i = 0; i < 16 / kWaves; ++i) {
      const int h = wave * (16 / kWaves) + i;
      copy16(a.q + (t * a.heads + min(h0 + h, a.heads - 1)) * kHeadDim + 8 * lane,
             lds + L::kWeights + L::kQPitch * h);
    }
  }
  // ... and, all of it there, take what each lane needs.
  __device__ __forceinline__ void read_q() {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      q[i] = as_bf16x8(lds_read<u32x4>(lds + L::kWeights + L::kQPitch * row + 256 * (i / 4) +
                                       64 * group + 16 * (i % 4)));
  }
  __device__ __forceinline__ void copy_table() const {
    const int32_t* const table = a.block_table + this->request() * a.bt_stride;
    if (a.max_blocks > kTableCache || a.topk == 0) return;
#pragma unroll
    for (int n = 0; n < kTableCache / 64 / kWaves; ++n) {
      const int c = 64 * (n * kWaves + wave);
      if (c < a.max_blocks) copy4(table + min(c + lane, a.max_blocks - 1), lds + L::kTable + 4 * c);
    }
  }

  // s in log2 units, -inf where bit i of `live` is off.
  __device__ __forceinline__ f32x4 scores(f32x4 acc, uint32_t live) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = (live >> i) & 1 ? acc[i] * a.scale_log2 : -INFINITY;
    return acc;
  }
  // The two weights of a pair of BF16.
  static __device__ __forceinline__ float both(uint32_t pair) {
    return u2f(pair << 16) + u2f(pair & 0xffff0000u);
  }
  // Against the new maximum `top`: O, and l and r with the sums that are against `own`.
  __device__ __forceinline__ void advance(float top, float own, float sum, float rsum) {
    if (__ballot(top != m) != 0) {
      const float f = step_down(m, top);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[i] *= f;
      l *= f;
      r *= f;
      m = top;
    }
    // (the sums are zero where own is -inf, and NaN stays NaN)
    const float f = own == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(own - top);
    l += sum * f;
    r += rsum * f;
  }

  // What the wave reads of its tile to score it.
  struct Tile {
    u32x4 code[4], scale;
    uint32_t bytes, live;
  };
  __device__ __forceinline__ void tile(int i, Tile& x) const {
    const uint32_t at = lds + (i & (kBuffers - 1)) * L::kRound + (wave >> 1) * kChunkBytes +
                        (wave & 1) * kTileBytes;
    const uint32_t rec = at + row * kMx4RecordBytes;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.code[j] = lds_read<u32x4>(rec + 64 * j + 16 * group);
    x.scale = lds_read<u32x4>(rec + kMx4CodeBytes);
    // lane c of a group: scale byte c of the group's four records
    const i32x2 two = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(lds_void*)(uintptr_t)(
        at + (4 * group + ((row >> 1) & 3)) * kMx4RecordBytes + kMx4CodeBytes + 8 * (row & 1)));
    x.bytes = (uint32_t)two[0];
    x.live = lds_read<uint32_t>(lds + L::kLive +
                                4 * ((i & (kBuffers - 1)) * L::kChunks + (wave >> 1))) >>
             (16 * (wave & 1) + 4 * group);
  }
  // Round i's weights, scale exponents and reference of the wave's tile, to LDS. between():
  // run behind the product, when the tile's registers are free.
  template <class F>
  __device__ __forceinline__ void score(int i, const Tile& x, const F& between) {
    const uint32_t chunk = (i & 1) * L::kChunks + (wave >> 1);
    f32x4 acc[2] = {zero_f(), zero_f()};
    uint32_t byte[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) byte[j] = (x.scale[j] >> (8 * group)) & 0xffu;
    // A scale past the reference would wrap the weights' exponents: NaN, as for 255 (four
    // instructions a tile; times unchanged, 256 tokens x 2,048 records 45.2 us and 45.4)
    if (max(max(byte[0], byte[1]), max(byte[2], byte[3])) > kScaleRef) byte[3] = kMx4NanScale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f = mx4_scale(byte[j]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        acc[u & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            as_bf16x8(fp4x8_to_bf16(x.code[j][u], f)), q[4 * j + u], acc[u & 1], 0, 0, 0);
    }
    u32x2 shift;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t two = __builtin_amdgcn_perm(0, x.bytes, k ? 0x0c030c02u : 0x0c010c00u);
      const u16x2 down = u16x2{kScaleRef, kScaleRef} - __builtin_bit_cast(u16x2, two);
      shift[k] = __builtin_bit_cast(uint32_t, (u16x2)(down << 7));
    }
    lds_write(lds + L::kShifts + 1024 * chunk + 64 * row + 16 * group + 8 * (wave & 1), shift);
    __builtin_amdgcn_sched_barrier(0);
    between();
    __builtin_amdgcn_sched_barrier(0);
    const f32x4 s = scores(acc[0] + acc[1], x.live);
    const float top = over_groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    const float own = top > m + kSlack ? ceilf(top) : m;
    const float ref = own == -INFINITY ? 0.0f : own;
    if (__ballot(own != m) != 0 && lane == 0) lds_write(lds + L::kMoved + 4 * (i & 3), 1);
    owns = own;
    float p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = __builtin_amdgcn_exp2f(s[k] - ref);
    sums = (p[0] + p[1]) + (p[2] + p[3]);
    const u32x2 pb = {__builtin_bit_cast(uint32_t, bf16_pair(p[0], p[1])),
                      __builtin_bit_cast(uint32_t, bf16_pair(p[2], p[3]))};
    rsums = both(pb[0]) + both(pb[1]);
    lds_write(lds + L::kWeights + 1024 * chunk + 16 * lane + 8 * (wave & 1), pb);
    if (lane < 16) lds_write(lds + L::kTops + 64 * ((i & 1) * kWaves + wave) + 4 * lane, own);
  }
  // A tile that the round does not have: weights of zero.
  __device__ __forceinline__ void no_score(int i) {
    const uint32_t chunk = (i & 1) * L::kChunks + (wave >> 1);
    owns = -INFINITY;
    sums = rsums = 0.0f;
    lds_write(lds + L::kWeights + 1024 * chunk + 16 * lane + 8 * (wave & 1), u32x2{0, 0});
    if (lane < 16) lds_write(lds + L::kTops + 64 * ((i & 1) * kWaves + wave) + 4 * lane, -INFINITY);
  }

  // What the wave reads of a chunk for its coordinates: the weights, and by group (32
  // coordinates) the scale exponents and codes.
  struct Operands {
    u32x4 shift;
    i32x2 v;
  };
  // By chunk c at w_at + 1024 c, s_at + 1024 c + 64 b and v_at + kChunkBytes c + 16 b.
  struct Places {
    uint32_t w_at, s_at, v_at;
  };
  __device__ __forceinline__ Places places(int i) const {
    const uint32_t odd = (i & 1) * 1024 * L::kChunks;
    return {lds + L::kWeights + odd + 16 * lane,
            lds + L::kShifts + odd + 64 * wave * (kTiles / 2) + 16 * group,
            lds + (i & (kBuffers - 1)) * L::kRound + ((row >> 2) & 1) * kTileBytes +
                (4 * group + (row & 3)) * kMx4RecordBytes + 8 * (row >> 3) + 16 * wave * (kTiles / 2)};
  }
  __device__ __forceinline__ void operands(const Places& at, int c, int b, Operands& x) const {
    x.shift = lds_read<u32x4>(at.s_at + 1024 * c + 64 * b);
    x.v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
        (lds_i32x2*)(lds_void*)(uintptr_t)(at.v_at + kChunkBytes * c + 16 * b));
  }
  // A chunk's weights against the running maximum; of0, of1: its tiles' references.
  __device__ __forceinline__ void lower(u32x4& p, float of0, float of1) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // whole log2 units down to the maximum, in both exponents; 255: past every exponent,
      // also for a tile without a record (of -inf, and the difference perhaps NaN)
      const uint32_t down = __umul24((uint32_t)fminf(m - (k ? of1 : of0), 255.0f), 0x00800080u);
      p[2 * k] = sub_sat(p[2 * k], down);
      p[2 * k + 1] = sub_sat(p[2 * k + 1], down);
    }
  }
  // O of group b of the wave's coordinates += a chunk.
  __device__ __forceinline__ void values(int b, const u32x4& p, const Operands& x) {
    u32x4 pw;
#pragma unroll
    for (int i = 0; i < 4; ++i) pw[i] = sub_sat(p[i], x.shift[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      o[2 * b + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          as_bf16x8(fp4x8_to_bf16((uint32_t)x.v[i], 1.0f)), as_bf16x8(pw), o[2 * b + i], 0, 0, 0);
  }

  // O += a round, whose first chunk's operands are p and y. kMoved: the tiles' references
  // `of` are not all the running maximum. kLast: the round has `here` chunks.
  template <bool kMoved, bool kLast>
  __device__ __forceinline__ void add(const Places& at, const float (&of)[kWaves], u32x4 (&p)[2],
                                      Operands (&y)[2], int here) {
    constexpr int kGroups = kTiles / 2, kSteps = L::kChunks * kGroups;
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      const int c = n / kGroups, b = n % kGroups, next = n + 1;
      if (kLast && b == 0 && c > 0 && c >= here) break;
      if (next < kSteps) {
        if (next % kGroups == 0) p[(c + 1) & 1] = lds_read<u32x4>(at.w_at + 1024 * (c + 1));
        operands(at, next / kGroups, next % kGroups, y[next & 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (kMoved && b == 0) lower(p[c & 1], of[2 * c], of[2 * c + 1]);
      values(b, p[c & 1], y[n & 1]);
    }
  }

  // Between two barriers: scores of round i (but after the last), O += round i - 1 (but
  // before the first). before: whether round i - 2 moved the maximum, since when round i -
  // 1 was scored without knowing.
  template <bool kFirst, bool kLast>
  __device__ __forceinline__ void step(int i, bool& before) {
    Operands y[2];
    u32x4 p[2];
    int moved = 0;
    const float own = owns, sum = sums, rsum = rsums;
    const Places at = places(i - 1);
    auto ahead = [&] {
      if (kFirst) return;
      moved = lds_read<int>(lds + L::kMoved + 4 * ((i - 1) & 3));
      p[0] = lds_read<u32x4>(at.w_at);
      operands(at, 0, 0, y[0]);
    };
    if (kLast) {
      ahead();
    } else if (i * L::kChunks + (wave >> 1) < this->chunks) {
      Tile x;
      tile(i, x);
      __builtin_amdgcn_sched_barrier(0);
      score(i, x, ahead);
    } else {
      ahead();
      no_score(i);
    }
    if (!kLast && threadIdx.x == 0) lds_write(lds + L::kMoved + 4 * ((i + 2) & 3), 0);
    if (kFirst) return;
    const bool now = uniform(moved) != 0;
    const int here = kLast ? this->chunks - (i - 1) * L::kChunks : L::kChunks;
    float of[kWaves];
    if (now || before) {
      float top = m;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        of[w] = lds_read<float>(lds + L::kTops + 64 * (((i - 1) & 1) * kWaves + w) + 4 * row);
        top = fmaxf(top, of[w]);
      }
      advance(top, own, sum, rsum);
      add<true, kLast>(at, of, p, y, here);
    } else {
      l += sum;
      r += rsum;
      add<false, kLast>(at, of, p, y, here);
    }
    before = now;
  }
  // The share of the list: chunk c of the split's is number c * splits + split.
  __device__ __forceinline__ void list() {
    bool before = false;
    step<true, false>(0, before);
    lds_barrier();
    for (int i = 1; i < this->rounds; ++i) {
      step<false, false>(i, before);
      lds_barrier();
    }
    step<false, true>(this->rounds, before);
  }

  // The window: chunks of 16 rows.
  __device__ __forceinline__ int window_entry(int first) const { return 16 * (first + wave) + row; }
  __device__ __forceinline__ void window() {
    const int32_t* const swa = a.swa_indices + t * a.swa_topk;
    const uint32_t at = lds + wave * kWindowBytes;
    for (int first = 0; first < this->back; first += kWaves) {
      const int waves = min(this->back - first, kWaves);
      float own = -INFINITY, sum = 0.0f, rsum = 0.0f;
      lds_barrier();
      if (wave < waves) {
        const int k = window_entry(first);
        int64_t slot = first == 0 ? lds_read<int>(lds + L::kEarly + 64 * wave + 4 * row)
                       : k < this->rows ? swa[k] : -1;
        if (k >= this->rows) slot = -1;
        const bool ok = slot >= 0 && slot < a.swa_rows;
        const uint8_t* page = a.swa_pool + (ok ? slot >> 6 : 0) * kNativePageBytes;
        const int in_page = ok ? (int)(slot & 63) : 0;
        const uint8_t* data = page + in_page * kNativeDataBytes;
        const uint32_t mask = (uint32_t)__ballot(ok) & 0xffffu;
#pragma unroll
        for (int j = 0; j < 9; ++j) copy16(data + 64 * j + 16 * group, at + 1024 * j);
        u32x2 srow = *(const u32x2*)(page + kPageRecords * kNativeDataBytes + in_page * kScaleBytes);
        wait_copies<0>();
        // A row that is no entry becomes zeros: its bytes could be codes or scales of NaN.
        if (!ok) {
#pragma unroll
          for (int j = 0; j < 9; ++j) lds_write(at + 1024 * j + 16 * lane, u32x4{0, 0, 0, 0});
          srow = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
        }
        srow[1] = (srow[1] & 0x00ffffffu) | 0x7f000000u;  // the tail has no scale
#pragma unroll
        for (int i = 0; i < 2; ++i)  // [64-coordinate group][row]
          lds_write<uint8_t>(at + kWindowScalesAt + 16 * (2 * group + i) + row,
                             (uint8_t)(srow[group >> 1] >> (16 * (group & 1) + 8 * i)));
        wave_lds_sync();
        f32x4 acc[2] = {zero_f(), zero_f()};
        auto piece = [&](int n) { return at + 1024 * (n >> 2) + 256 * (n & 3) + 16 * row; };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = u2f(((srow[j / 2] >> (16 * (j % 2) + 8 * (group >> 1))) & 0xffu) << 23);
          // coordinates 128 j + 32 group: codes, or (448 and up) the BF16 tail
          const bool tail = j == 3 && group >= 2;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const u32x4 c16 = lds_read<u32x4>(piece(tail ? 28 + 4 * (group - 2) + u
                                                         : 8 * j + 2 * group + u / 2));
            const uint32_t lo = c16[2 * (u % 2)], hi = c16[2 * (u % 2) + 1];
            u32x4 k8 = {fp8_pair_to_bf16<false>(lo, f), fp8_pair_to_bf16<true>(lo, f),
                        fp8_pair_to_bf16<false>(hi, f), fp8_pair_to_bf16<true>(hi, f)};
            if (j == 3) k8 = tail ? c16 : k8;
            acc[u & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(k8), q[4 * j + u],
                                                                 acc[u & 1], 0, 0, 0);
          }
        }
        const f32x4 s = scores(acc[0] + acc[1], mask >> (4 * group));
        own = ceilf(over_groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
        const float ref = own == -INFINITY ? 0.0f : own;
        f32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = __builtin_amdgcn_exp2f(s[i] - ref);
          sum += p[i];
        }
        rsum = both(__builtin_bit_cast(uint32_t, bf16_pair(p[0], p[1]))) +
               both(__builtin_bit_cast(uint32_t, bf16_pair(p[2], p[3])));
        lds_write(lds + L::kWeights + 1024 * wave + 16 * lane, __builtin_bit_cast(u32x4, p));
        if (lane < 16) lds_write(lds + L::kTops + 64 * wave + 4 * lane, own);
      }
      lds_barrier();
      float top = m;
#pragma unroll 1
      for (int w = 0; w < waves; ++w)
        top = fmaxf(top, lds_read<float>(lds + L::kTops + 64 * w + 4 * row));
      advance(top, own, sum, rsum);
#pragma unroll 1
      for (int w = 0; w < waves; ++w) {
        const uint32_t from = lds + w * kWindowBytes;
        const float own_w = lds_read<float>(lds + L::kTops + 64 * w + 4 * row);
        // (O is in units of 2^32)
        const float f = own_w == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(own_w - m - 32.0f);
        f32x4 p = lds_read<f32x4>(lds + L::kWeights + 1024 * w + 16 * lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] *= f;
        // 32 coordinates (two tiles) a turn: codes below 448, the BF16 tail above
#pragma unroll
        for (int b = 0; b < kTiles / 2; ++b) {
          const int g = wave * (kTiles / 2) + b;
          s16x4 v[2];
          if (32 * g < kNopeDim) {
            const int x = 32 * g + 16 * (row >> 3) + 8 * (row & 1);
            const uint32_t src = from + 1024 * (x >> 6) + 256 * ((x >> 4) & 3) +
                                 16 * (4 * group + ((row >> 1) & 3)) + (x & 8);
            const i32x2 c8 =
                __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(lds_void*)(uintptr_t)src);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              v[i] = __builtin_bit_cast(s16x4, u32x2{fp8_pair_to_bf16<false>((uint32_t)c8[i], 1.0f),
                                                     fp8_pair_to_bf16<true>((uint32_t)c8[i], 1.0f)});
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int x = kNopeDim + 2 * (32 * g - kNopeDim + 16 * i) + 8 * (row & 3);
              const uint32_t src = from + 1024 * (x >> 6) + 256 * ((x >> 4) & 3) +
                                   16 * (4 * group + (row >> 2)) + (x & 8);
              v[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)(uintptr_t)src);
            }
          }
          const uint32_t bytes = lds_read<uint32_t>(from + kWindowScalesAt + 16 * (g / 2) + 4 * group);
          f32x4 pw;
#pragma unroll
          for (int i = 0; i < 4; ++i) pw[i] = p[i] * u2f(((bytes >> (8 * i)) & 0xffu) << 23);
          const s16x4 pb = __builtin_bit_cast(
              s16x4, u32x2{__builtin_bit_cast(uint32_t, bf16_pair(pw[0], pw[1])),
                           __builtin_bit_cast(uint32_t, bf16_pair(pw[2], pw[3]))});
#pragma unroll
          for (int i = 0; i < 2; ++i)
            o[2 * b + i] =
                __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v[i], pb, o[2 * b + i], 0, 0, 0);
        }
      }
      lds_barrier();
    }
  }

  __device__ __forceinline__ void finish() {
    l = over_groups_sum(l);
    r = over_groups_sum(r);
    lds_barrier();
    if (lane < 16) lds_write(lds + L::kTops + 128 * wave + 8 * lane, f32x2{l, r});
    lds_barrier();
    float sum = 0.0f, rsum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const f32x2 of = lds_read<f32x2>(lds + L::kTops + 128 * w + 8 * row);
      sum += of[0];
      rsum += of[1];
    }
    const int h = h0 + row;
    if (h >= a.heads) return;
    const int c0 = wave * kTiles * 16 + 4 * group;
    if (a.ws_splits != 0) {
      const int64_t at = ((int64_t)blockIdx.y * a.ws_splits + split) * a.heads + h;
      const float f = sum != 0.0f ? 0x1p32f * __builtin_amdgcn_rcpf(rsum) : 0.0f;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        __builtin_nontemporal_store(o[i] * f, (f32x4*)(a.ws_o + at * kHeadDim + c0 + 16 * i));
      // (NaN goes on as infinity: the combine's maximum would pass over a NaN)
      if (wave == 0 && lane < 16)
        a.ws_lse[at] = sum != sum     ? INFINITY
                       : sum != 0.0f ? m + __builtin_amdgcn_logf(sum)
                                     : -INFINITY;
      return;
    }
    // (the sums are in normal range: the hardware's log2, exp2 and reciprocal, each within
    // an ulp, need no scaling)
    const float sink2 = a.sink ? a.sink[h] * kLog2e : -INFINITY;
    const float top = fmaxf(m, sink2);
    float f = 0.0f, lse = -INFINITY;
    if (top != -INFINITY || sum != 0.0f) {
      const float em = m == -INFINITY && sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
      const float z = sum * em + __builtin_amdgcn_exp2f(sink2 - top);
      // (O over the rounded weights' sum, times the list's share of z)
      if (sum != 0.0f)
        f = 0x1p32f * __builtin_amdgcn_rcpf(rsum) * (sum * em * __builtin_amdgcn_rcpf(z));
      lse = (top + __builtin_amdgcn_logf(z)) * kLn2;
    }
    if (wave == 0 && lane < 16) a.lse[t * a.heads + h] = lse;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const f32x4 v = o[i] * f;
      *(u32x2*)(a.out + (t * a.heads + h) * kHeadDim + c0 + 16 * i) =
          u32x2{__builtin_bit_cast(uint32_t, bf16_pair(v[0], v[1])),
                __builtin_bit_cast(uint32_t, bf16_pair(v[2], v[3]))};
    }
  }
};

template <int kWaves>
__global__ __launch_bounds__(96 * kWaves) void mx4_decode_kernel(DecodeArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Lds<kWaves>::kBytes];
  const uint32_t at = (uint32_t)(uintptr_t)(lds_void*)lds;
  if (threadIdx.x >= 64 * kWaves) {  // (s_barrier counts the waves that have not ended)
    Copier<kWaves>(a, at).run();
    return;
  }
  Decode<kWaves> d(a, at);
  d.copy_table();
  d.copy_q();
  int early = -1;
  if (a.swa_topk > 0)
    early = a.swa_indices[d.t * a.swa_topk + min(d.window_entry(0), a.swa_topk - 1)];
  d.lengths();
  // (kept in LDS: the list's loop needs the registers)
  if (a.swa_topk > 0) lds_write(at + Lds<kWaves>::kEarly + 64 * d.wave + 4 * d.row, early);
  wait_copies<0>();
  lds_barrier();
  d.read_q();
  if (threadIdx.x == 0) lds_write(at + Lds<kWaves>::kMoved, u32x2{0, 0});
  lds_barrier();
  if (d.rounds > 0) d.list();
  if (d.back > 0) d.window();
  d.finish();
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

bool bad_sizes(int64_t tokens, int64_t heads, int64_t topk, int64_t swa_topk) {
  return tokens < 0 || tokens > 65535 || heads < 0 || heads > kMaxHeads || topk < 0 ||
         topk > kMaxTopk || swa_topk < 0 || swa_topk > kMaxWindow;
}

constexpr int kWaves = 8;  // that compute, a workgroup

struct Plan {
  int64_t alone;  // tokens with one workgroup a 16 heads
  int slots;      // workgroups a 16 heads of each of the others
  int splits;     // of them the list's; the window, where there is one, has the last
};

// At most one workgroup a CU (256; its LDS allows one at a time), so that all run at once:
// 96 tokens x 2,048 records 29.4 us with two a token and 44.1 with three, 129 tokens 40.0
// with one and 52.4 with two. No more than the rounds divide by (43 tokens x 16 rounds: 20.8
// us with four a token, 21.5 with five), and one alone where splitting saves a round only,
// which the second kernel costs again (32 tokens x 2 rounds 9.4 and 10.2 us, x 3 rounds 12.4
// and 10.9; 1 token x 2 rounds 9.0 both); with more tokens their partial results count too
// (96 tokens x 4 rounds 15.5 and 16.0). The window's rows are fetched while the list's are
// where it has a workgroup to itself.
// Beyond 256 workgroups it is the tokens of the last, partial turn that are split, in a
// launch of their own (270 tokens x 2,048 records 78.7 -> 59.4 us, 300 79.5 -> 68.2, 384
// 83.4 -> 79.3, 520 118.8 -> 100.6; 384 x 512 34.8 both; one launch for both kinds took 2.5
// less there and 0.2 more on one token, 9.2).
Plan plan(int64_t tokens, int64_t heads, int64_t topk, int64_t swa_topk) {
  const int64_t groups = std::max<int64_t>((heads + 15) / 16, 1);
  const int64_t rounds = (topk + 16 * kWaves - 1) / (16 * kWaves), window = swa_topk > 0;
  const int64_t alone = tokens * groups / 256 * 256 / groups;
  const int64_t base = std::max<int64_t>((tokens - alone) * groups, 1);
  const int64_t most = std::min({256 / base - window, rounds, kMaxSplits - window});
  if (alone == tokens || most < 1) return {tokens, 1, 1};
  const int64_t each = (rounds + most - 1) / most;
  if (64 * (rounds + window - std::max(each, window)) < 64 + base) return {tokens, 1, 1};
  const int64_t splits = (rounds + each - 1) / each;
  return {alone, (int)(splits + window), (int)splits};
}
size_t ws_bytes(const Plan& p, int64_t tokens, int64_t heads) {
  return (size_t)((tokens - p.alone) * p.slots * heads) * (kHeadDim + 1) * sizeof(float);
}

}  // namespace

extern "C" int rm_mx4_sparse_decode_workspace(int64_t tokens, int64_t heads, int64_t topk,
                                              int64_t swa_topk, int32_t* num_splits,
                                              size_t* workspace_bytes) {
  if (bad_sizes(tokens, heads, topk, swa_topk)) return RM_ERR_SHAPE;
  const Plan p = plan(tokens, heads, topk, swa_topk);
  if (num_splits) *num_splits = p.slots;
  if (workspace_bytes) *workspace_bytes = ws_bytes(p, tokens, heads);
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
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(pool, 16) || !aligned(swa_pool, 16))
    return RM_ERR_ALIGN;
  for (const void* p : {(const void*)block_table, (const void*)seqlens, (const void*)indices,
                        (const void*)topk_length, (const void*)swa_indices,
                        (const void*)swa_length, (const void*)sink, (const void*)lse})
    if (!aligned(p, 4)) return RM_ERR_ALIGN;
  const Plan p = plan(tokens, heads, topk, swa_topk);
  const size_t bytes = ws_bytes(p, tokens, heads);
  if (bytes > 0 && (!workspace || workspace_bytes < bytes)) return RM_ERR_WORKSPACE;
  if (bytes > 0 && !aligned(workspace, 16)) return RM_ERR_ALIGN;
  DecodeArgs a;
  a.q = q;
  a.q_len_magic = (((uint64_t)1 << 32) + q_len - 1) / q_len;
  a.heads = (int)heads;
  a.pool = pool;
  a.pool_pages = (int)pool_pages;
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.max_blocks = (int)max_blocks;
  a.seqlens = seqlens;
  a.indices = indices;
  // (an entry that is none reads the pool's first record: without one the list is empty)
  a.topk = pool_pages > 0 && max_blocks > 0 ? (int)topk : 0;
  a.once = tokens * topk * kMx4RecordBytes >= kOnceBytes;
  a.topk_length = topk_length;
  a.swa_pool = swa_pool;
  a.swa_rows = swa_pool_pages * kPageRecords;
  a.swa_indices = swa_indices;
  a.swa_topk = swa_pool_pages > 0 ? (int)swa_topk : 0;
  a.swa_length = swa_length;
  a.sink = sink;
  a.scale_log2 = softmax_scale * kLog2e;
  a.out = out;
  a.lse = lse;
  hipStream_t s = (hipStream_t)stream;
  const unsigned groups = (unsigned)((heads + 15) / 16);
  if (p.alone > 0) {
    a.first = 0;
    a.splits = 1;
    a.splits_magic = (uint64_t)1 << 32;
    a.window_split = a.ws_splits = 0;
    a.ws_o = a.ws_lse = nullptr;
    hipLaunchKernelGGL(mx4_decode_kernel<kWaves>, dim3(1, (unsigned)p.alone, groups),
                       dim3(96 * kWaves), 0, s, a);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  const int64_t rest = tokens - p.alone;
  if (rest > 0) {
    a.first = (int)p.alone;
    a.splits = a.window_split = p.splits;
    a.splits_magic = (((uint64_t)1 << 32) + p.splits - 1) / p.splits;
    a.ws_splits = p.slots;
    a.ws_o = (float*)workspace;
    a.ws_lse = (float*)workspace + (size_t)rest * p.slots * heads * kHeadDim;
    hipLaunchKernelGGL(mx4_decode_kernel<kWaves>, dim3((unsigned)p.slots, (unsigned)rest, groups),
                       dim3(96 * kWaves), 0, s, a);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
    launch_combine<true>(a.ws_o, a.ws_lse, sink, p.slots, rest, heads,
                         out + p.alone * heads * kHeadDim, lse + p.alone * heads, s);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  return RM_OK;
}
