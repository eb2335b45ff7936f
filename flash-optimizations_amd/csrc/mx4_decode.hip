// Sparse-MLA decode over 4-bit records, jointly with sliding-window rows of a
// Native pool. For query token t and head h, over the valid entries j of t's list
// and window (K_j the dequantized 512-coordinate row, V = K):
//   l_j = (q_h . K_j) * scale, Z = sum_j exp(l_j) + exp(sink_h),
//   out = sum_j exp(l_j) K_j / Z, lse = ln Z.
//
// A workgroup of kWaves waves owns (split of a list, token, 16 heads) and walks its
// share in rounds of 32 records a wave. A round has two halves with a barrier
// between:
//   * scores: a wave holds its 32 records as the A operands of S^T = K Q^T
//     (v_mfma_f32_16x16x32_bf16; lane (r, g) loads 64 contiguous code bytes of
//     record r straight from its row, four scale groups, so Q, in registers, is
//     ordered to match). It leaves in LDS the raw code bytes, the weights P
//     = 2^(s - m) as BF16, m = ceil of its 32 scores' maximum, and each record's
//     scale exponents.
//   * values: a wave owns 512 / kWaves output coordinates of O^T += V^T P^T over
//     all the round's records. The codes come out of LDS transposed
//     (ds_read_b64_tr_b4: 8 records of 32 coordinates a lane pair) and become BF16
//     without their scales; the scales are powers of two that differ by record and
//     group, so they go to the weights instead, and so does the step from the
//     wave's m to the running maximum: an integer subtraction on the BF16
//     exponents, two weights an instruction, saturating at zero (v_pk_sub_u16
//     clamp), against the largest scale the store writes, 2^32; O is in units of it.
//     A weight that a scale takes below 2^-126 becomes zero: less than 2^-71 of the
//     largest weight at that scale.
// Both operands keep the order of the score tile: P^T in LDS is what the lane
// holding it writes, 16 bytes a lane, with no exchange between lanes.
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
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

struct DecodeArgs {
  const uint16_t* q;
  int q_len, heads;
  const uint8_t* pool;
  int pool_pages;
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
  int splits;     // of the list; workgroup x = splits takes the window rows
  int ws_splits;  // partial slots a row; 0: finish in place
  uint16_t* out;
  float* lse;
  float* ws_o;    // [tokens, ws_splits, heads, 512]
  float* ws_lse;  // [tokens, ws_splits, heads]
};

// A round's data of one wave. Codes: two tiles of 16 records, 272 bytes apart (4
// banks), the second tile half a bank row off, so that the transposed reads of a
// lane group's 2 x 4 records meet no bank twice.
constexpr int kCodePitch = 272;
constexpr int kTileBytes = 16 * kCodePitch + 128;
// Window rows: 16 a wave, the 576 data bytes 592 apart.
constexpr int kRowPitch = 592;
constexpr int kScaleRef = 127 + kMx4MaxExponent;

struct WaveLds {
  union {
    struct {
      uint8_t codes[2 * kTileBytes];
      uint16_t shift[16][32];  // [group][record slot]: (159 - scale byte) << 7
    };
    struct {
      uint8_t rows[16 * kRowPitch];
      uint8_t scales[8][16];   // [group][row]
    };
  };
  u32x4 weight[64];            // by lane; a list: 8 BF16, a window: 4 floats
  float top[16];               // by head: the exponent the weights are against
};

__device__ __forceinline__ float over_groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float over_groups_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
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

// 2^(from - to) for running maxima, 1 where both are -inf (nothing yet).
__device__ __forceinline__ float step_down(float from, float to) {
  return from == to ? 1.0f : exp2f(from - to);
}

template <int kWaves>
struct Decode {
  static constexpr int kTiles = kHeadDim / 16 / kWaves;  // 16-coordinate tiles of O a wave
  const DecodeArgs& a;
  WaveLds* const lds;  // [kWaves]
  const int lane, wave, row, group;  // row: record of a tile, or head; group: lane / 16
  const int64_t t;
  const int h0;
  bf16x8 q[16];     // q[4 j + u]: coordinates 128 group + 32 j + 8 u .. + 7 of head `row`
  f32x4 o[kTiles];  // coordinate 16 tile + 4 group + i of head `row`
  float m, l;       // running maximum of head `row` (whole log2 units); this lane's sum

  __device__ __forceinline__ Decode(const DecodeArgs& args, WaveLds* sm)
      : a(args),
        lds(sm),
        lane(wave_lane()),
        wave(uniform((int)(threadIdx.x >> 6))),
        row(lane & 15),
        group(lane >> 4),
        t(blockIdx.y),
        h0(blockIdx.z * 16) {
    const uint16_t* src = a.q + (t * a.heads + min(h0 + row, a.heads - 1)) * kHeadDim + 128 * group;
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = as_bf16x8(*(const u32x4*)(src + 8 * i));
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.0f;
  }

  // Weights of one score tile's four records: against `ref`, zero where bit i of
  // `live` is off.
  __device__ __forceinline__ f32x4 scores(f32x4 acc, uint32_t live) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = (live >> i) & 1 ? acc[i] * a.scale_log2 : -INFINITY;
    return acc;
  }
  // The round's running maximum, from what the waves left; rescales O and l.
  __device__ __forceinline__ void advance(int waves, float own, float sum) {
    float top = m;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (w < waves) top = fmaxf(top, lds[w].top[row]);
    const float f = step_down(m, top);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i] *= f;
    // (sum is zero where own is -inf, and NaN stays NaN)
    l = l * f + (own == -INFINITY ? sum : sum * exp2f(own - top));
    m = top;
  }

  // The list's records [begin, end).
  __device__ __forceinline__ void list(int begin, int end) {
    const int64_t request = t / a.q_len;
    const int32_t* const idx = a.indices + t * a.topk;
    const int32_t* const table = a.block_table + request * a.bt_stride;
    const int records = a.seqlens ? a.seqlens[request] : 0x7fffffff;
    WaveLds& mine = lds[wave];
    for (int at = begin; at < end; at += 32 * kWaves) {
      const int waves = min((end - at + 31) / 32, kWaves);
      float own = -INFINITY, sum = 0.0f;
      if (wave < waves) {
        f32x4 s[2];
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          const int k = at + 32 * wave + 16 * tile + row;
          const int r = k < end ? idx[k] : -1;
          const int column = r >> 6;
          const bool inside = r >= 0 && r < records && column < a.max_blocks;
          const int page = inside ? table[column] : -1;
          const bool live = page >= 0 && page < a.pool_pages;
          const int64_t slot = live ? (int64_t)page * kPageRecords + (r & 63) : 0;
          const uint8_t* rec = a.pool + slot * kMx4RecordBytes;
          u32x4 code[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) code[j] = *(const u32x4*)(rec + 64 * group + 16 * j);
          const uint32_t scale = *(const uint32_t*)(rec + kMx4CodeBytes + 4 * group);
          const uint32_t mask = (uint32_t)__ballot(live) & 0xffffu;
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
          uint8_t* const dst = mine.codes + tile * kTileBytes + row * kCodePitch + 64 * group;
          const int rslot = 8 * (row >> 2) + 4 * tile + (row & 3);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *(u32x4*)(dst + 16 * j) = code[j];
            const uint32_t byte = (scale >> (8 * j)) & 0xffu;
            mine.shift[4 * group + j][rslot] = (uint16_t)((kScaleRef - byte) << 7);
            const float f = mx4_scale(byte);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(fp4x8_to_bf16(code[j][u], f)),
                                                            q[4 * j + u], acc, 0, 0, 0);
          }
          s[tile] = scores(acc, mask >> (4 * group));
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(s[0][i], s[1][i]));
        own = ceilf(over_groups_max(top));
        const float ref = own == -INFINITY ? 0.0f : own;
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = exp2f(s[i / 4][i % 4] - ref);
          sum += p[i];
        }
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_bit_cast(uint32_t, bf16_pair(p[2 * i], p[2 * i + 1]));
        mine.weight[lane] = w;
        if (lane < 16) mine.top[lane] = own;
      }
      lds_barrier();
      advance(waves, own, sum);
#pragma unroll 1
      for (int w = 0; w < waves; ++w) {
        const WaveLds& from = lds[w];
        const float own_w = from.top[row];
        // (255: past every exponent)
        const int down = own_w == -INFINITY ? 255 : (int)fminf(m - own_w, 255.0f);
        u32x4 p = from.weight[lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = sub_sat(p[i], (uint32_t)down * 0x00800080u);
        const uint8_t* codes = from.codes + ((row >> 2) & 1) * kTileBytes +
                               (4 * group + (row & 3)) * kCodePitch + 8 * (row >> 3);
#pragma unroll
        for (int b = 0; b < kTiles / 2; ++b) {
          const int g = wave * (kTiles / 2) + b;
          const u32x4 shift = *(const u32x4*)&from.shift[g][8 * group];
          u32x4 pw;
#pragma unroll
          for (int i = 0; i < 4; ++i) pw[i] = sub_sat(p[i], shift[i]);
          const i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)(lds_void*)(codes + 16 * g));
#pragma unroll
          for (int i = 0; i < 2; ++i)
            o[2 * b + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                as_bf16x8(fp4x8_to_bf16((uint32_t)v[i], 1.0f)), as_bf16x8(pw), o[2 * b + i], 0, 0, 0);
        }
      }
      lds_barrier();
    }
  }

  // The token's window rows [0, end), 16 a wave and round.
  __device__ __forceinline__ void window(int end) {
    const int32_t* const idx = a.swa_indices + t * a.swa_topk;
    WaveLds& mine = lds[wave];
    for (int at = 0; at < end; at += 16 * kWaves) {
      const int waves = min((end - at + 15) / 16, kWaves);
      float own = -INFINITY, sum = 0.0f;
      if (wave < waves) {
        const int k = at + 16 * wave + row;
        const int64_t slot = k < end ? idx[k] : -1;
        const bool live = slot >= 0 && slot < a.swa_rows;
        const uint8_t* page = a.swa_pool + (live ? slot >> 6 : 0) * kNativePageBytes;
        const int in_page = live ? (int)(slot & 63) : 0;
        const uint8_t* data = page + in_page * kNativeDataBytes;
        const uint32_t mask = (uint32_t)__ballot(live) & 0xffffu;
        // The lane's 128 coordinates: 128 codes, or (group 3) 64 codes and the tail. A row
        // that is no entry becomes zeros: its bytes could be codes or scales of NaN.
        u32x4 code[8], tail[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          code[c] = *(const u32x4*)(data + 128 * group + 16 * (group == 3 ? c & 3 : c));
          tail[c] = *(const u32x4*)(data + kNopeDim + 16 * c);
        }
        const u32x2 srow =
            *(const u32x2*)(page + kPageRecords * kNativeDataBytes + in_page * kScaleBytes);
        const u32x4 zero = {0, 0, 0, 0};
        uint8_t* const dst = mine.rows + row * kRowPitch;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          code[c] = live ? code[c] : zero;
          tail[c] = live ? tail[c] : zero;
          if (group < 3 || c < 4) *(u32x4*)(dst + 128 * group + 16 * c) = code[c];
          if (group == 3) *(u32x4*)(dst + kNopeDim + 16 * c) = tail[c];
        }
        const uint32_t sbytes = live ? srow[group >> 1] >> (16 * (group & 1)) : 0x7f7fu;
        mine.scales[2 * group][row] = (uint8_t)sbytes;
        mine.scales[2 * group + 1][row] = group == 3 ? 127 : (uint8_t)(sbytes >> 8);  // (tail: none)
        f32x4 acc = zero_f();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = u2f(((sbytes >> (8 * (j / 2))) & 0xffu) << 23);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const u32x4 c = code[2 * j + u / 2];
            const uint32_t lo = c[2 * (u % 2)], hi = c[2 * (u % 2) + 1];
            u32x4 k8 = {fp8_pair_to_bf16<false>(lo, f), fp8_pair_to_bf16<true>(lo, f),
                        fp8_pair_to_bf16<false>(hi, f), fp8_pair_to_bf16<true>(hi, f)};
            if (j >= 2) k8 = group == 3 ? tail[4 * (j - 2) + u] : k8;
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(k8), q[4 * j + u], acc, 0, 0, 0);
          }
        }
        const f32x4 s = scores(acc, mask >> (4 * group));
        own = ceilf(over_groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
        const float ref = own == -INFINITY ? 0.0f : own;
        f32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = exp2f(s[i] - ref);
          sum += p[i];
        }
        mine.weight[lane] = __builtin_bit_cast(u32x4, p);
        if (lane < 16) mine.top[lane] = own;
      }
      lds_barrier();
      advance(waves, own, sum);
#pragma unroll 1
      for (int w = 0; w < waves; ++w) {
        const WaveLds& from = lds[w];
        const float own_w = from.top[row];
        const float f = own_w == -INFINITY ? 0.0f : exp2f(own_w - m);
        f32x4 p = __builtin_bit_cast(f32x4, from.weight[lane]);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] *= f;
        // 32 coordinates (two tiles) a turn: codes below 448, the BF16 tail above
#pragma unroll
        for (int b = 0; b < kTiles / 2; ++b) {
          const int c0 = 32 * (wave * (kTiles / 2) + b);
          s16x4 v[2];
          if (c0 < kNopeDim) {
            const uint8_t* src = from.rows + (4 * group + ((row >> 1) & 3)) * kRowPitch + c0 +
                                 16 * (row >> 3) + 8 * (row & 1);
            const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(lds_void*)src);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t lo = fp8_pair_to_bf16<false>((uint32_t)c[i], 1.0f);
              const uint32_t hi = fp8_pair_to_bf16<true>((uint32_t)c[i], 1.0f);
              v[i] = __builtin_bit_cast(s16x4, u32x2{lo, hi});
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint8_t* src = from.rows + (4 * group + (row >> 2)) * kRowPitch + kNopeDim +
                                   2 * (c0 - kNopeDim + 16 * i + 4 * (row & 3));
              v[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_void*)src);
            }
          }
          const uint32_t bytes = *(const uint32_t*)&from.scales[c0 / 64][4 * group];
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
  static __device__ __forceinline__ f32x4 zero_f() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

  // unit: what O is in units of.
  __device__ __forceinline__ void finish(int slot, float unit) {
    l = over_groups_sum(l);
    if (lane < 16) lds[wave].top[lane] = l;
    lds_barrier();
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += lds[w].top[row];
    const int h = h0 + row;
    const bool write = h < a.heads;
    const int c0 = wave * kTiles * 16 + 4 * group;
    if (a.ws_splits != 0) {
      const int64_t at = (t * a.ws_splits + slot) * a.heads + h;
      const float f = sum != 0.0f ? unit / sum : 0.0f;
      if (!write) return;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
        __builtin_nontemporal_store(o[i] * f, (f32x4*)(a.ws_o + at * kHeadDim + c0 + 16 * i));
      // (NaN goes on as infinity: the combine's maximum would pass over a NaN)
      if (wave == 0 && lane < 16)
        a.ws_lse[at] = sum != sum ? INFINITY : sum != 0.0f ? m + log2f(sum) : -INFINITY;
      return;
    }
    const float sink2 = a.sink && write ? a.sink[h] * kLog2e : -INFINITY;
    const float top = fmaxf(m, sink2);
    float f = 0.0f, lse = -INFINITY;
    if (top != -INFINITY || sum != 0.0f) {
      const float em = m == -INFINITY && sum == 0.0f ? 0.0f : exp2f(m - top);
      const float z = sum * em + exp2f(sink2 - top);
      f = em * unit / z;
      lse = (top + log2f(z)) * kLn2;
    }
    if (!write) return;
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
__global__ __launch_bounds__(64 * kWaves) void mx4_decode_kernel(DecodeArgs a) {
  __shared__ __attribute__((aligned(16))) WaveLds lds[kWaves];
  Decode<kWaves> d(a, lds);
  if ((int)blockIdx.x < a.splits) {
    int live = a.topk;
    if (a.topk_length) live = max(min(a.topk_length[d.t], live), 0);
    // consecutive shares of whole 32-record tiles
    const int share = ((live + a.splits - 1) / a.splits + 31) & ~31;
    const int begin = min((int)blockIdx.x * share, live);
    d.list(begin, min(begin + share, live));
    d.finish(blockIdx.x, 0x1p32f);
  } else {
    int live = a.swa_topk;
    if (a.swa_length) live = max(min(a.swa_length[d.t], live), 0);
    d.window(live);
    d.finish(blockIdx.x, 1.0f);
  }
}

bool aligned(const void* p, uintptr_t al) { return ((uintptr_t)p & (al - 1)) == 0; }

bool bad_sizes(int64_t tokens, int64_t heads, int64_t topk, int64_t swa_topk) {
  return tokens < 0 || tokens > 65535 || heads < 0 || heads > kMaxHeads || topk < 0 ||
         topk > kMaxTopk || swa_topk < 0 || swa_topk > kMaxWindow;
}

struct Plan {
  int waves;   // a workgroup
  int splits;  // of the list (0: no list)
  int slots;   // partial slots a row: the splits and the window rows' workgroup
};

// About one workgroup of eight waves a CU (256): enough splits to reach that, each
// with a full round of records.
Plan plan(int64_t tokens, int64_t heads, int64_t topk, int64_t swa_topk) {
  Plan p;
  p.waves = 8;
  const int64_t base = std::max<int64_t>(tokens * ((heads + 15) / 16), 1);
  const int64_t rounds = (topk + 32 * p.waves - 1) / (32 * p.waves);
  int64_t splits = (256 + base - 1) / base;
  splits = std::min({splits, rounds, (int64_t)kMaxSplits - 1});
  p.splits = (int)std::max<int64_t>(splits, topk > 0 || swa_topk == 0 ? 1 : 0);
  p.slots = p.splits + (swa_topk > 0 ? 1 : 0);
  return p;
}
size_t ws_bytes(int64_t tokens, int64_t heads, int64_t slots) {
  return slots > 1 ? (size_t)(tokens * slots * heads) * (kHeadDim + 1) * sizeof(float) : 0;
}

}  // namespace

extern "C" int rm_mx4_sparse_decode_workspace(int64_t tokens, int64_t heads, int64_t topk,
                                              int64_t swa_topk, int32_t* num_splits,
                                              size_t* workspace_bytes) {
  if (bad_sizes(tokens, heads, topk, swa_topk)) return RM_ERR_SHAPE;
  const Plan p = plan(tokens, heads, topk, swa_topk);
  if (num_splits) *num_splits = p.slots;
  if (workspace_bytes) *workspace_bytes = ws_bytes(tokens, heads, p.slots);
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
  const Plan p = plan(tokens, heads, topk, swa_topk);
  const size_t bytes = ws_bytes(tokens, heads, p.slots);
  if (bytes > 0 && (!workspace || workspace_bytes < bytes)) return RM_ERR_WORKSPACE;
  if (bytes > 0 && !aligned(workspace, 16)) return RM_ERR_ALIGN;
  DecodeArgs a;
  a.q = q;
  a.q_len = (int)q_len;
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
  a.topk_length = topk_length;
  a.swa_pool = swa_pool;
  a.swa_rows = swa_pool_pages * kPageRecords;
  a.swa_indices = swa_indices;
  a.swa_topk = swa_pool_pages > 0 ? (int)swa_topk : 0;
  a.swa_length = swa_length;
  a.sink = sink;
  a.scale_log2 = softmax_scale * kLog2e;
  a.splits = p.splits;
  a.ws_splits = p.slots > 1 ? p.slots : 0;
  a.out = out;
  a.lse = lse;
  a.ws_o = (float*)workspace;
  a.ws_lse = bytes ? (float*)workspace + (size_t)tokens * p.slots * heads * kHeadDim : nullptr;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)p.slots, (unsigned)tokens, (unsigned)((heads + 15) / 16));
  hipLaunchKernelGGL(mx4_decode_kernel<8>, grid, dim3(64 * p.waves), 0, s, a);
  if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  if (p.slots > 1) {
    launch_combine<true>(a.ws_o, a.ws_lse, sink, p.slots, tokens, heads, out, lse, s);
    if (hipGetLastError() != hipSuccess) return RM_ERR_LAUNCH;
  }
  return RM_OK;
}
