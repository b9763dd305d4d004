// Attention over the quantised key / value cache, for the newest few tokens of each sequence (decoding).
//
// Mathematics.  A row's value is zero_g + scale_g * code for the channels of group g (int4), scale * code (e4m3).  With the
// codes of 16 tokens as the 16-row operand of a 16 x 8 x 16 MMA and up to eight query rows (the q heads of a kv head, times
// the tokens of the call) as its columns,
//   S[t, r] = sum_g scale_g[t] * (sum_{d in g} code[t, d] q[r, d]) + zero_g[t] * (sum_{d in g} q[r, d])
//   O[d, r] = sum_t code[t, d] * (P[t, r] scale_g[t]) + sum_t P[t, r] zero_g[t],        P = exp2(S * c - m[r])
// so no code is ever multiplied by its scale: the products run on codes, scales enter S by sums over a group and O by way
// of P.  Both products and all sums are fp32; q, P * scale and the codes are f16:
//   * a code 0 .. 15 in the low bits of a half IS a number of f16, code * 2^-24 (a subnormal, exact, which MMAs take at
//     full speed), and in the next four bits 16 times that.  Unpacking eight codes to four f16 pairs is four ANDs and a
//     shift; the 2^24 and the 16 are powers of two that go into the row's factor, q and the result.
//   * q is scaled by a power of two for each row so that its largest entry is near 2^14: bf16 and f16 values lose at most
//     bits that are 2^-24 of that entry.
//   * P * scale is scaled by a power of two for each row, below 2^14: 11 bits of it are kept, though nothing below 2^-22 of the row's
//     largest (a row's largest stands at 2^-3 at least, and f16 ends at 2^-25).  The power follows the largest scale seen, or the
//     row's largest P * scale where that is far less: values of a key without weight, however large, cost the others nothing.  What
//     remains: where the scales of one row's groups of channels are 2^11 apart and more, the smaller group keeps fewer bits than 11.
//     That is enough for outputs of bf16 (1.73e-3 of the norm from 64 bits where rounding the output alone costs 1.64e-3).  For
//     f16 what is left of it goes through a second product, and int4's codes are taken less 8, with 8 scale_g in the zeros: sums
//     of codes, all positive, are far larger than what comes out of long and even rows, and their own rounding in 32 bits shows.
//     f16, int4, 5111 and 60000 keys: 6.0e-4 without either, 2.4e-4 and 4.7e-4 with the second product, 2.0e-4 and 2.2e-4
//     with both, where rounding the output costs 2.0e-4 (e4m3: 2.8e-4, 2.1e-4 with the second product).  It costs a
//     sixth: 32 sequences of 8192 .. 32768, 32 / 8 heads of 128, bf16 150 us, f16 179.  Codes less 8 are not left as subnormals: MMAs
//     line up products by the exponents that their factors are written with, and cut off up to 2^-15 of a product of a subnormal.
//   * sums of int4 codes are levelled every kLevelTokens tokens of a warp, see there: their error does not grow with the call.
// Softmax statistics are of one pass over the keys, with a running maximum and sum for each row.
//
// Split: the keys of all (sequence, kv head, row tile) items, one after the other in units of kUnit tokens, are cut into
// equal shares for the CTAs, wherever that falls in a sequence.  A share is found on the device from the lengths: the host
// never needs them, and the launch can be captured in a graph.  The warps of a CTA take the units of its share of an
// item in turn, each with a ring of its own in shared memory (cp.async; no barrier between warps while keys stream), and
// put their sums together at the end of the item.  An item that more than one CTA has worked on is joined by a second kernel,
// from sums in the workspace, in the order of the CTAs: results do not depend on who comes first.  Where sequences cannot be long
// every item is one CTA's, and there is one launch.
// Page tables by kv head and query (chosen pages) are of much the same length: an item is shared by the CTAs of a cluster, which put
// their sums together in their shared memory, in the order of the CTAs, again without a second launch (form_by_head).
//
// Bound by: no one thing.  HBM asks for 64 + 8 bytes a token, head and side (int4, head dim 128, groups of 64), 46 codes a cycle and SM at
// 6.5 TB/s; a warp spends some 545 instructions on a unit of 32 tokens (keys and values, eight rows; 160 of them unpack), 2.2 for
// 32 codes, and an SM issues 2.2 a cycle of the 4 that it could, its 14 warps waiting for their own last instruction most often.  The
// copies alone, with the products left out, take most of the time as well (us of a call, whole : copies alone; 32 / 8 heads of 128,
// int4): 32 sequences of 8192 .. 32768 149.9 : 119.9, one of 131072 41.4 : 35.0, 64 of 200 .. 4096 48.8 : 38.0: copies, first loads
// and launches bound a call as much as its instructions do, and warps that wait at one of them do not get on with the other.
// Throughput 4.9, 3.6 and 3.4 TB/s of the 6.5 that a plain copy reaches.  About 9 us of each call are the two launches and the chains of
// loads at their beginnings (lengths, pages, codes; parts).  e4m3 rows are unpacked by conversions and ask for twice the bytes: 48
// sequences of 0 .. 13025 109 us, 6.2 TB/s.
// Rows of more than one block of eight spend 190 instructions more a block on a unit, and leave room for fewer warps.  Registers: the
// element type is a value at run time, so a kernel holds four forms of the product with P (masked or not, f16's second product or
// not); 34 of the 50 kernels spill, up to 224 bytes a thread (most where groups of 32 keep many scales), the forms that are timed here
// 0 (e4m3) to 36 (head dim 64 in groups of 32).
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>

#include "cache_common.cuh"

namespace sb {

// Warps of a CTA; kMostWarps where every item is one CTA's and there are fewer than two for an SM (us, 4 : 8 warps, up to 1024
// tokens, 8 items 12.5 : 10.6, 256 items 14.6 : 14.6, 1024 items 35.6 : 44.3; tables by head: form_by_head).  Shares: four CTAs of 4
// warps on an SM and two of 8 are alike where sequences are long, short ones want the smaller CTAs (64 x 200 .. 4096: 53.6 : 56.3).
constexpr int kWarps = 4, kMostWarps = 8;
constexpr int kMostCluster = 8;

struct AttendParams {
  const uint8_t* k_codes;
  const uint8_t* k_scales;
  const uint8_t* v_codes;
  const uint8_t* v_scales;
  const void* q;
  void* o;
  const int32_t* page_table;
  const int32_t* lengths;
  float* lse;
  float* max_logits;
  const float* sinks;
  // workspace: for each CTA two items it may share with others, sums [rows][row_v], then max and sum [2][rows]
  float* parts;
  int64_t* starts;  // [batch + 1] where each sequence's items begin, in the measure of shares
  int64_t q_stride_b, q_stride_h, q_stride_s, o_stride_b, o_stride_h, o_stride_s, table_stride, n_pages;
  float scale, soft_cap, mask_value;
  // A page table is of a sequence, or (by head) of a sequence, kv head and query: `batch` counts tables, q_len is 1 then, and
  // `queries` is what q has of them.  items: kv heads of a table times row tiles.
  int32_t batch, q_heads, kv_heads, heads_per_kv, q_len, queries, items, row_tiles, n_table, page_size, page_shift, dtype;
  int32_t head_dim, head_dim_v, window, item_cost;  // item_cost: in units
  int32_t cluster;  // whole: CTAs of a cluster that share an item
  bool whole;       // every item is one CTA's, or one cluster's
};

// ------------------------------------------------------------------------------------------
// instructions
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldmatrix_x2(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x2_trans(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A word's codes 0 and 4 (odd: 1 and 5) less 8, as a pair of halves that are no subnormals: 1024 + code and 64 + code have a code in
// just the bits where it stands.  Exact.  (The mask and the exponent in one instruction, which the compiler does not find: f16, 32 x
// 8192 .. 32768 tokens 194 -> 179 us.)
__device__ __forceinline__ uint32_t less_eight(uint32_t word, bool odd) {
  uint32_t pair;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;"  // (a & b) | c
      : "=r"(pair)
      : "r"(word), "r"(odd ? 0x00f000f0u : 0x000f000fu), "r"(odd ? 0x54005400u : 0x64006400u));
  const uint32_t less = odd ? 0xd480d480u : 0xe408e408u;  // -72, -1032
  const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&pair), *reinterpret_cast<const __half2*>(&less));
  return *reinterpret_cast<const uint32_t*>(&x);
}

// ------------------------------------------------------------------------------------------
// sizes
// ------------------------------------------------------------------------------------------
// kK, kV: padded widths of a row; kG: channels of a group (int4); kN: blocks of eight query rows
template <int kFormat_, int kK_, int kV_, int kG_, int kN_>
struct AttendShape {
  static constexpr int kFormat = kFormat_, kK = kK_, kV = kV_, kN = kN_;
  static constexpr bool kInt4 = kFormat == SPLASH_CACHE_INT4;
  static_assert(kN >= 1 && kN <= 3);
  static constexpr int kRows = 8 * kN;
  static constexpr int kRowK = cache_row_bytes(kFormat, kK), kRowV = cache_row_bytes(kFormat, kV);
  // Tokens of a unit.  A warp has a unit in flight while it works on another: about 4 KB (a quarter more or less with what 16
  // tokens are), which fills the shared memory of an SM with 16 warps.  Where the rows' sums leave registers for 8 or 12 warps,
  // a unit may be 8 KB (e4m3, head dim 128, 24 rows, 16 sequences of 1000 .. 8192 tokens: 63 -> 60 us), unless the logits
  // of 32 tokens do not fit beside the sums (int4, whose scales take registers too).
  static constexpr int kRowBytes = kRowK + kRowV;
  static constexpr int kUnit = kN > 2   ? (kInt4 ? (kRowBytes <= 64 ? 32 : 16) : kRowBytes <= 256 ? 32 : 16)
                               : kN == 2 ? (kRowBytes <= (kInt4 ? 128 : 256) ? 32 : 16)
                                         : (kRowBytes <= 64 ? 64 : kRowBytes <= 128 ? 32 : 16);
  static constexpr int kTiles = kUnit / 16;
  // channels that 16 bytes of codes hold, and MMA steps (16 channels) over them
  static constexpr int kChunk = kInt4 ? 32 : 16, kSteps = kChunk / 16;
  static constexpr int kGroupsK = kInt4 ? kK / kG_ : 1, kGroupsV = kInt4 ? kV / kG_ : 1;
  static constexpr int kChunksK = kK / kChunk, kChunksV = kV / kChunk;
  static constexpr int kPerGroupK = kChunksK / kGroupsK, kPerGroupV = kChunksV / kGroupsV;
  static constexpr int kScaleK = cache_scale_bytes(kFormat, kK, kG_), kScaleV = cache_scale_bytes(kFormat, kV, kG_);
  static constexpr int kStageBytes = (kUnit * (kRowK + kRowV + kScaleK + kScaleV) + 127) / 128 * 128;
  static constexpr int kRegisters = kV * kN / 4 + 90;  // sums, and about what else a thread holds
  static constexpr int kResident = 65536 / (kWarps * 32 * (kRegisters < 128 ? 128 : kRegisters));  // CTAs of an SM
  static constexpr int kMostRegisters = kResident >= 4 ? 128 : kResident == 3 ? 168 : 255;
  // shared memory
  static constexpr int kFragBytes = kK / 16 * kN * 256;            // q as fragments
  static constexpr int kQSums = kFragBytes;                        // [kGroupsK][kRows] sums of q over a group
  static constexpr int kFactors = kQSums + kGroupsK * kRows * 4;   // [kRows] what S is multiplied by
  static constexpr int kStats = kFactors + kRows * 4;              // [3][kMostWarps][kRows] of the warps, see there
  static constexpr int kRing = (kStats + 3 * kMostWarps * kRows * 4 + 127) / 128 * 128;
  // of a warp: its two stages, and in their place its sums [kRows][kV] once they have run dry
  static constexpr int kWarpBytes = 2 * kStageBytes > kRows * kV * 4 ? 2 * kStageBytes : kRows * kV * 4;
  __host__ __device__ static constexpr int smem(int warps) { return kRing + warps * kWarpBytes; }
  static constexpr int smem_cluster(int warps) { return smem(warps) + (kRows * kV / 8 + kMostCluster) * 48; }  // (sums of a cluster's CTAs)
};

// Where in a stage 16-byte piece c of row r lies: so that eight consecutive rows' piece c are in eight different bank groups.
// The low bits of c, those in kTurn, are turned by the row.
template <int kRowBytes>
struct Pieces {
  static constexpr int kEach = kRowBytes / 16;
  static constexpr int kTurn = kEach % 8 == 0 ? 7 : kEach % 4 == 0 ? 3 : kEach % 2 == 0 ? 1 : 0;
  static constexpr int kShift = kEach % 8 == 0 ? 0 : kEach % 4 == 0 ? 1 : 2;
  static __device__ __forceinline__ int row_at(int r) { return r * kRowBytes + ((r >> kShift & kTurn) << 4); }
  // `row`: the address of row_at() in an area that starts at a multiple of 128
  static __device__ __forceinline__ uint32_t at(uint32_t row, int c) { return (row ^ ((c & kTurn) << 4)) + ((c & ~kTurn) << 4); }
};

// Sixteen rows of the tile at `place` to `to` (a multiple of 128), 16 bytes a lane and step.
template <int kRowBytes>
__device__ __forceinline__ void copy_rows(uint32_t to, const uint8_t* codes, uint32_t place, int lane) {
  using P = Pieces<kRowBytes>;
  const uint8_t* const from = codes + ((uint64_t)place * (16 * kRowBytes) + lane * 16);
  constexpr bool kAlike = 32 % P::kEach == 0 && 32 / P::kEach % 8 == 0;  // every step's rows are turned alike
  const uint32_t first = to + P::at(P::row_at(lane / P::kEach), lane % P::kEach);
#pragma unroll
  for (int j = 0; j < (kRowBytes + 31) / 32; ++j) {
    const int piece = j * 32 + lane;
    const uint32_t at = kAlike ? first + j * 512 : to + P::at(P::row_at(piece / P::kEach), piece % P::kEach);
    if (kRowBytes % 32 == 0 || piece < kRowBytes) cp_async16(at, from + j * 512);
  }
}

// A 16-byte piece of the rows of kTiles tiles: words of rows g and g + 8.  `at`: this lane's row of the first two tiles.
template <int kTiles, int kRowBytes>
__device__ __forceinline__ void load_tiles(uint32_t at, uint32_t (&words)[kTiles][2]) {
  if constexpr (kTiles == 1) {
    ldmatrix_x2(at, words[0][0], words[0][1]);
  } else {
#pragma unroll
    for (int i = 0; i < kTiles; i += 2) ldmatrix_x4(at + i * 16 * kRowBytes, words[i][0], words[i][1], words[i + 1][0], words[i + 1][1]);
  }
}

// kCount consecutive words of shared memory, kCount * 4 bytes from a multiple of that times any number.
template <int kCount>
__device__ __forceinline__ void load_words(uint32_t (&w)[kCount], const uint32_t* from) {
  if constexpr (kCount % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(from + i);
      w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
    }
  } else if constexpr (kCount % 2 == 0) {
#pragma unroll
    for (int i = 0; i < kCount; i += 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(from + i);
      w[i] = x.x, w[i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i) w[i] = from[i];
  }
}

constexpr float kNoMaximum = -1.0e30f;  // of a row that has seen no key yet: finite, so that differences are
constexpr float kSlack = 8.f;           // how far (in units of log2) logits may pass the maximum that P is taken against
constexpr float kUnitLog2 = 5.f;        // P * scale is below 2^(kSlack + 1 + kUnitLog2) = 2^14
// Tokens of a warp after which the sums of int4 codes are levelled (bf16, 32 / 8 heads of 128, us with 512, 768, 1024 and never: 32 x
// 8192 .. 32768 tokens 151.7, 150.7, 150.0, 147.5; one of 131072, 41.6, 41.7, 41.4, 41.4; relative error of outputs over even rows of
// 131072 and 2^20 tokens, in calls of 1.3e8 and 1e8 of them: 512 1.8e-3 and 2.8e-3, 1024 1.9e-3 and 3.4e-3, never 4.5e-2 and 0.16).
constexpr int kLevelTokens = 1024;
constexpr uint32_t kLeastTop = 87u << 23;  // 2^-40
constexpr float kCodeUnit = 0x1p24f;  // a code in the low bits of a half, in units of the number that it is there
constexpr float kLeastTopLog2 = -40.f, kSpare = 8.f, kRoom = 6.f;

// ------------------------------------------------------------------------------------------
// shares
// ------------------------------------------------------------------------------------------
// What a CTA spends on an item beside its units, in tokens: shares are equal in the sum of both.  (Looking up the item, q as
// fragments, the first keys' latency, the warps' sums together: some thousand cycles, more with more rows.)  us with 160, 320, 480, 640 and
// 960 tokens, int4 | e4m3:
//   8 rows of 128    64 x 200 .. 4096, 8 kv heads      53.6 49.6 50.5 50.6 52.8 | 60.4 60.1 61.0 62.1 65.2
//   8 rows of 256    24 x 300 .. 9000, 4               37.9 37.9 38.3 39.3 40.4 | 45.6 46.2 46.0 45.9 45.8
//   16 rows of 64    24 x 300 .. 8000, 4               29.2 27.3 27.1 27.1 27.8 | 29.1 27.3 27.0 27.0 28.1
//   16 rows of 128   32 x 200 .. 6000, 4               37.5 34.7 34.2 34.2 36.3 | 39.4 36.1 34.9 35.0 36.1
//   16 of 192 / 128  24 x 300 .. 9000, 4               43.8 41.4 42.0 42.8 44.4 | 46.5 43.4 43.4 44.2 45.6
//   16 rows of 256   32 x 8000 .. 30000, 2             124.2 121.2 120.5 121.1 122.4 | 119.9 117.1 118.4 119.4 119.9
//   20 rows of 128   16 x 1000 .. 8192, 8              64.6 59.9 59.9 60.1 62.2 | 54.9 52.6 49.7 49.8 51.6
__host__ __device__ constexpr int item_tokens(int blocks) { return blocks == 1 ? 320 : 480; }
// Every item is one CTA's where queries see at most kWholeTokens, or twice as many and there are kWholeItems .. kMostWholeItems - 1
// items (us, whole : shares and a second launch; 1024 tokens, 8 items 10.5 : 11.5, 256 items 14.6 : 18.8, 1024 items 35.0 : 37.9;
// 2048 tokens, 8 items 14.6 : 11.6, 64 items 14.9 : 14.7, 256 items 22.6 : 24.9, 1024 items 57.4 : 52.8; 3000 tokens, 256 items
// 28.3 : 27.6).
constexpr int kWholeTokens = 1024, kWholeItems = 64, kMostWholeItems = 4 * kSms;

struct Keys {  // of a sequence: tokens [lo, hi) in whole units from lo, which is a multiple of kUnit
  int lo, hi, units;
  __device__ int cost(const AttendParams& p) const { return units > 0 ? units + p.item_cost : 0; }
};
template <int kUnit>
__device__ __forceinline__ Keys keys_of(const AttendParams& p, int length) {
  Keys k;
  const int64_t reach = (int64_t)p.n_table << p.page_shift;
  k.hi = (int)min((int64_t)max(length, 0), reach);
  k.lo = p.window < 0 ? 0 : max((int)max((int64_t)length - p.q_len - p.window, (int64_t)0), 0) / kUnit * kUnit;
  k.units = k.lo < k.hi ? (k.hi - k.lo + kUnit - 1) / kUnit : 0;
  return k;
}

// a / b for a >= 0, b > 0; 32 bits wide where that is enough (a division of 64 bits takes some hundred cycles).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return (a | b) >> 32 == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ int64_t share_of(int64_t total, int ctas) {  // a unit for each warp at least
  const int64_t share = quotient(total + ctas - 1, ctas);
  return share > kWarps ? share : kWarps;
}

// (What a kernel of sequences' tables works out from other parameters it is not given again: the compiler finds other registers for it,
// and some calls take 1 to 3 % longer.)
template <bool kByHead>
__device__ __forceinline__ int items_of_table(const AttendParams& p) {
  return kByHead ? p.items : p.kv_heads * p.row_tiles;
}

struct Start {  // where a CTA's share begins
  int64_t total, before;  // cost of all items, and of those of the sequences before b
  int64_t share;
  int b;
};

// All threads of a CTA of kWarps; `scratch`: kWarps + 2 words of shared memory of 8 bytes.  Sequences go by the threads of a
// CTA at a time; a second look is taken only where there are more of them than that.
template <int kUnit, bool kByHead>
__device__ Start find_start(const AttendParams& p, int64_t* scratch) {
  constexpr int kThreads = kWarps * 32;
  const int64_t per_sequence = items_of_table<kByHead>(p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t* const found = scratch + kWarps;
  const bool keep = blockIdx.x == 0;  // this CTA writes down where the sequences start
  const bool once = p.batch <= kThreads;
  int64_t total = 0, share = 0, at = 0;
  for (int look = once ? 1 : 0; look < 2; ++look) {
    int64_t carry = 0;
    for (int base = 0; base < p.batch; base += kThreads) {
      const int b = base + tid;
      const int64_t mine = b < p.batch ? keys_of<kUnit>(p, __ldg(p.lengths + b)).cost(p) * per_sequence : 0;
      int64_t sum = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t other = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += other;
      }
      if (base > 0 || look > 0) __syncthreads();  // (before what the last round left is written over)
      if (lane == 31) scratch[warp] = sum;
      __syncthreads();
      int64_t before = carry + sum - mine;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int64_t s = scratch[w];
        before += w < warp ? s : 0;
        carry += s;
      }
      if (look == 1) {
        if (once) {
          total = carry;
          share = share_of(total, gridDim.x);
          at = blockIdx.x * share;
        }
        if (b < p.batch) {
          if (keep) p.starts[b] = before;
          if (at >= before && at < before + mine) {
            found[0] = b;
            found[1] = before;
          }
        }
      }
    }
    if (look == 0) {
      total = carry;
      share = share_of(total, gridDim.x);
      at = blockIdx.x * share;
    }
  }
  if (keep && tid == 0) p.starts[p.batch] = total;
  __syncthreads();
  return {total, found[1], share, (int)found[0]};
}

// ------------------------------------------------------------------------------------------
// the kernel
// ------------------------------------------------------------------------------------------
// What a row's sums become: the output row, or a part of it in the workspace.  `m` in units of log2, with the sink in it.
__device__ __forceinline__ void add_sink(float sink, float& m, float& l) {
  const float s = sink * kLog2e, top = fmaxf(m, s);
  l = l * ex2(m - top) + ex2(s - top);
  m = top;
}

// The sequence, kv head and first query of the rows of an item: table b, kv head times row tiles `item`.
struct Rows {
  int b, head, query;
};
template <bool kByHead>
__device__ __forceinline__ Rows rows_of(const AttendParams& p, int b, int item) {
  if constexpr (!kByHead) return {b, item / p.row_tiles, 0};
  const unsigned pair = (unsigned)b / (unsigned)p.queries;
  return {(int)(pair / (unsigned)p.kv_heads), (int)(pair % (unsigned)p.kv_heads), (int)((unsigned)b % (unsigned)p.queries)};
}

// Eight channels of a row, from the sums of all its keys.
template <bool kByHead>
__device__ __forceinline__ void finish_row(const AttendParams& p, const Rows& rows, int row, int d, float (&x)[8], float m, float l) {
  const int b = rows.b, i = rows.query + row / p.heads_per_kv, h = rows.head * p.heads_per_kv + row % p.heads_per_kv;
  float weight = 1.f;
  if (p.sinks != nullptr) {
    const float own = m;
    add_sink(__ldg(p.sinks + h), m, l);
    weight = ex2(own - m);
  }
  weight = l == 0.f ? 0.f : weight / l;
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] *= weight;
  if (d < p.head_dim_v) store8(p.o, p.dtype, b * p.o_stride_b + h * p.o_stride_h + i * p.o_stride_s + d, x);
  if (d == 0) {
    const int64_t to = ((int64_t)b * p.q_heads + h) * (kByHead ? p.queries : p.q_len) + i;
    if (p.lse != nullptr) p.lse[to] = l == 0.f ? p.mask_value : (m + __log2f(l)) * kLn2;
    if (p.max_logits != nullptr) p.max_logits[to] = l == 0.f ? p.mask_value : m * kLn2;
  }
}

// kByHead: a page table for each kv head and query.  (A kernel of its own: what it holds beside would cost the others registers, and 2 to
// 7 % of their time.)
template <typename Shape, bool kByHead>
__global__ void __maxnreg__(Shape::kMostRegisters) cache_attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kN = Shape::kN, kRows = Shape::kRows, kUnit = Shape::kUnit, kTiles = Shape::kTiles, kSteps = Shape::kSteps;
  constexpr int kGroupsK = Shape::kGroupsK, kGroupsV = Shape::kGroupsV;
  constexpr bool kInt4 = Shape::kInt4;
  extern __shared__ __align__(128) uint8_t smem[];
  float* const q_sums = reinterpret_cast<float*>(smem + Shape::kQSums);
  float* const factors = reinterpret_cast<float*>(smem + Shape::kFactors);
  // of each warp and row: the highest logit, what P was taken against, the sum of P (all as that leaves it)
  float* const warp_high = reinterpret_cast<float*>(smem + Shape::kStats);
  float* const warp_base = warp_high + kMostWarps * kRows;
  float* const warp_sum = warp_base + kMostWarps * kRows;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  if (!kByHead || !p.whole) grid_dependents_launch();  // the joining kernel may come up beside this one; it waits for its end
  if (kByHead) grid_dependency_wait();     // (where this one has come up beside the kernel that chose its pages)

  const int per_sequence = items_of_table<kByHead>(p);
  const bool clustered = kByHead && p.cluster > 1;
  const int rank = clustered ? blockIdx.x % (unsigned)p.cluster : 0;
  int64_t at, end, before, share_begin;  // in the measure of shares; before: what lies before sequence b
  int b;
  if (p.whole) {  // items in turn
    at = kByHead ? blockIdx.x / (unsigned)p.cluster : blockIdx.x;
    end = (int64_t)p.batch * per_sequence;
  } else {
    const Start start = find_start<kUnit, kByHead>(p, reinterpret_cast<int64_t*>(smem));
    __syncthreads();  // (its scratch is about to be q's place)
    at = share_begin = (int64_t)blockIdx.x * start.share;
    end = min(at + start.share, start.total);
    b = start.b;
    before = start.before;
  }
  uint8_t* const ring = smem + Shape::kRing + warp * Shape::kWarpBytes;
  // of a cluster: the sums of all its CTAs for the channels that this one finishes, [eight channels][CTA][eight sums, maximum, sum of P, 2]
  float* const received = reinterpret_cast<float*>(smem + Shape::smem(warps));
  if (clustered) cluster_arrive();
  const uint32_t ring_at = smem_u32(ring);
  const int heads = p.heads_per_kv;

  // The item that is worked on (or whose keys are on their way): b, item = head * row_tiles + row tile, units u0 .. u1 - 1.
  int item = 0, u0 = 0, u1 = 0, length = 0, head = 0;
  Keys keys{};
  bool is_last = false;  // its first unit is in this share, so that its sums are those of place 1
  auto next_item = [&]() -> bool {
    if (at >= end) return false;
    if (p.whole) {
      b = (int)((unsigned)at / (unsigned)per_sequence);
      item = (int)((unsigned)at % (unsigned)per_sequence);
      length = __ldg(p.lengths + b);
      if constexpr (kByHead) {  // (the length is on its way: see below)
        at += gridDim.x / (unsigned)p.cluster;
      } else {
        keys = keys_of<kUnit>(p, length);
        u0 = 0;
        u1 = keys.units;
        at += gridDim.x;
      }
    } else {
      length = __ldg(p.lengths + b);
      keys = keys_of<kUnit>(p, length);
      while (at >= before + (int64_t)keys.cost(p) * per_sequence) {  // (sequences without keys are passed over)
        before += (int64_t)keys.cost(p) * per_sequence;
        length = __ldg(p.lengths + ++b);
        keys = keys_of<kUnit>(p, length);
      }
      item = (int)quotient(at - before, keys.cost(p));
      const int64_t first = before + (int64_t)item * keys.cost(p) + p.item_cost;  // of its units
      u0 = (int)max(at - first, (int64_t)0);
      u1 = (int)min((int64_t)keys.units, end - first);
      is_last = first > share_begin;
      at = first + u1;
      if (u1 <= 0) return false;  // (the share ends before the item's keys)
    }
    return true;
  };

  // ---- keys on their way ----
  // Pages are looked up for kTurns of a warp's units at a time, a batch ahead: lane i has where tile i of the batch lies,
  // in tiles of the whole cache.
  constexpr uint32_t kNowhere = ~0u;
  constexpr int kTurns = 32 / kTiles;
  auto look_up = [&](int turn) -> uint32_t {
    const int u = u0 + warp + (turn + lane / kTiles) * warps, token = keys.lo + u * kUnit + lane % kTiles * 16;
    const int page = u < u1 && token < keys.hi ? __ldg(p.page_table + b * p.table_stride + (token >> p.page_shift)) : -1;
    if (page < 0 || page >= p.n_pages) return kNowhere;
    const uint32_t first = (uint32_t)(page * p.kv_heads + (kByHead ? head : item / p.row_tiles)) << (p.page_shift - 4);
    return first + ((token & (p.page_size - 1)) >> 4);
  };
  uint32_t places, next_places;
  uint32_t absent;  // a bit for each tile of the batch that has no page
  auto copy_tile = [&](uint32_t place, uint32_t to, int i) {
    const uint32_t to_v = to + kUnit * Shape::kRowK, to_scales = to_v + kUnit * Shape::kRowV;
    copy_rows<Shape::kRowK>(to + i * 16 * Shape::kRowK, p.k_codes, place, lane);
    copy_rows<Shape::kRowV>(to_v + i * 16 * Shape::kRowV, p.v_codes, place, lane);
    if (lane < Shape::kScaleK)
      cp_async16(to_scales + i * Shape::kScaleK * 16 + lane * 16, p.k_scales + ((uint64_t)place * (Shape::kScaleK * 16) + lane * 16));
    if (lane < Shape::kScaleV)
      cp_async16(to_scales + kUnit * Shape::kScaleK + i * Shape::kScaleV * 16 + lane * 16,
                 p.v_scales + ((uint64_t)place * (Shape::kScaleV * 16) + lane * 16));
  };
  // Starts the copies of the warp's unit number `turn`; called for each in turn.  Returns a bit for each of its tiles that
  // has no page (its keys are not seen).
  auto fetch = [&](int turn, int stage) -> uint32_t {
    const int first = turn % kTurns * kTiles;
    if (first == 0 && turn > 0) {
      places = next_places;
      absent = __ballot_sync(~0u, places == kNowhere);
      next_places = look_up(turn + kTurns);
    }
    const uint32_t missing = absent >> first & ((1u << kTiles) - 1);
    const uint32_t to = ring_at + stage * Shape::kStageBytes;
    if (missing == 0) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) copy_tile(__shfl_sync(~0u, places, first + i), to, i);
    } else if (u0 + warp + turn * warps < u1) {
      for (int i = 0; i < kTiles; ++i) {
        const uint32_t place = __shfl_sync(~0u, places, first + i);
        if (!(missing >> i & 1)) copy_tile(place, to, i);
      }
    }
    cp_async_commit();
    return missing;
  };
  uint32_t next_missing = 0;  // of the unit that is on its way
  auto start_item = [&]() {
    places = look_up(0);
    next_places = look_up(kTurns);
    absent = __ballot_sync(~0u, places == kNowhere);
    next_missing = fetch(0, 0);
  };

  while (next_item()) {
    const Rows rows = rows_of<kByHead>(p, b, item);
    if (kByHead) head = rows.head;
    const int row0 = item % p.row_tiles * kRows;
    const int n_rows = min(kRows, p.q_len * heads - row0);

    // ---- q's rows on their way: kLanes lanes (a power of two that holds the row's width / 8) a row ----
    // Row r of the tile is query (first_row + r) / heads behind first_query (r and heads are small: the quotient by a product
    // is exact), q head (first_row + r) % heads of the kv head.
    const int first_query = row0 / heads, first_row = row0 - first_query * heads;
    const float per_head = 1.f / (float)heads;
    auto query_of = [&](int r) { return (int)(((float)(first_row + r) + 0.5f) * per_head); };
    constexpr int kLanes = Shape::kK <= 64 ? 8 : Shape::kK <= 128 ? 16 : 32, kAtOnce = 32 / kLanes;
    const int piece = lane % kLanes;
    constexpr int kPasses = (kRows + kWarps * kAtOnce - 1) / (kWarps * kAtOnce);  // (at most)
    uint4 raw[kPasses];
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      const int r = (pass * warps + warp) * kAtOnce + lane / kLanes;
      raw[pass] = make_uint4(0, 0, 0, 0);
      if (r < n_rows && piece * 8 < p.head_dim) {
        const int i = query_of(r), h = rows.head * heads + first_row + r - i * heads;
        raw[pass] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + rows.b * p.q_stride_b + h * p.q_stride_h +
                                                         (rows.query + first_query + i) * p.q_stride_s + piece * 8));
      }
    }
    if (kByHead && p.whole) {
      keys = keys_of<kUnit>(p, length);
      u0 = 0;
      u1 = keys.units;
      if (clustered) {
        u0 = keys.units * rank / p.cluster;  // (units are below 2^26)
        u1 = keys.units * (rank + 1) / p.cluster;
      }
    }
    start_item();

    // ---- and as fragments ----
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      const int r = (pass * warps + warp) * kAtOnce + lane / kLanes;
      if (pass * warps * kAtOnce >= kRows) break;  // (all warps alike)
      float x[8];
      unpack16(p.dtype, raw[pass].x, x[0], x[1]);
      unpack16(p.dtype, raw[pass].y, x[2], x[3]);
      unpack16(p.dtype, raw[pass].z, x[4], x[5]);
      unpack16(p.dtype, raw[pass].w, x[6], x[7]);
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) top = max3(top, fabsf(x[i]), fabsf(x[i + 1]));
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      // the power of two that brings `top` to 2^14 .. 2^15, within 2^-100 .. 2^100; with the sign of the logits' scale
      const int e = min(max((int)(__float_as_uint(top) >> 23), 41), 227);
      const float up = copysignf(__uint_as_float((uint32_t)(268 - e) << 23), p.scale), down = __uint_as_float((uint32_t)(e - 14) << 23);
      __half h16[8];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h16[i] = __float2half_rn(x[i] * up);
        if (kInt4) sum += __half2float(h16[i]);
      }
      auto two = [&](int lo, int hi) { return (uint32_t)__half_as_ushort(h16[lo]) | (uint32_t)__half_as_ushort(h16[hi]) << 16; };
      auto sixteenth = [&](uint32_t pair) {  // int4: the odd codes of a half-word stand four bits higher
        const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&pair), __float2half2_rn(0.0625f));
        return *reinterpret_cast<const uint32_t*>(&y);
      };
      if (r < kRows && piece * 8 < Shape::kK) {
        // For each 32 channels, block of rows and lane of the MMA: its part of both steps.
        uint4* const frag = reinterpret_cast<uint4*>(smem) + ((piece >> 2) * kN + (r >> 3)) * 32 + (r & 7) * 4;
        if (kInt4) {  // a lane's eight channels are one word of codes, column piece % 4
          const uint32_t odd = sixteenth(two(1, 5)), odd2 = sixteenth(two(3, 7));
          frag[piece & 3] = make_uint4(two(0, 4), odd, two(2, 6), odd2);
        } else {  // two words of codes: columns 2 * (piece % 2) and the next of step piece / 2 % 2
          uint2* const half = reinterpret_cast<uint2*>(frag + (piece & 1) * 2) + (piece >> 1 & 1);
          half[0] = make_uint2(two(0, 1), two(2, 3));
          half[2] = make_uint2(two(4, 5), two(6, 7));
        }
      }
      if (kInt4) {
        constexpr int kGroupLanes = Shape::kPerGroupK * 4;
#pragma unroll
        for (int d = 1; d < kGroupLanes; d <<= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if (r < kRows && piece % kGroupLanes == 0 && piece * 8 < Shape::kK)
          q_sums[piece / kGroupLanes * kRows + r] = sum * 0x1p-24f;  // in the units of the products of codes
      }
      // (not 0, so that logits of -inf keep being that)
      if (r < kRows && piece == 0)
        factors[r] = fmaxf(fabsf(p.scale) * down * (kInt4 ? 0x1p24f : 1.f) * (p.soft_cap > 0.f ? 1.f : kLog2e), 1e-37f);
    }
    __syncthreads();

    // ---- this lane's columns: rows nb * 8 + t4 * 2 and the next ----
    // highest: of this lane's logits; limit: what they may reach before the maximum is raised
    float limit[kN][2], base[kN][2], l[kN][2], factor[kN][2], highest[kN][2];
    float o[Shape::kChunksV][kSteps][kN][4] = {};
    float zeros[kGroupsV][kN][2] = {};
    // Each row's P is taken in units of a power of two throughout (in l, the zeros' sums and O; `base` has it), 2^kUnitLog2 over the
    // row's top: the largest scale of V seen, or 2^kRoom times the largest P * scale of the row where that is less by 2^kSpare,
    // which a key of huge values and no weight would otherwise leave few bits of.  As bits, rounded down to powers of two (2^-40 at
    // least): the least of the rows' tops, and the largest scale seen.
    uint32_t top = kLeastTop, largest_seen = kLeastTop;
#pragma unroll
    for (int nb = 0; nb < kN; ++nb)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        limit[nb][j] = base[nb][j] = highest[nb][j] = kNoMaximum;
        l[nb][j] = 0.f;
        factor[nb][j] = p.soft_cap > 0.f ? 1.f : factors[nb * 8 + t4 * 2 + j];
      }
    // units of which every row sees every key: whole_lo .. whole_hi - 1
    const int position0 = length - p.q_len + first_query;  // of the tile's first query
    const int whole_hi = (min(position0 + 1, keys.hi) - keys.lo) / kUnit;
    const int whole_lo = p.window < 0 ? 0 : max(position0 + query_of(n_rows - 1) - p.window - keys.lo + kUnit - 1, 0) / kUnit;

    const uint4* const frags = reinterpret_cast<const uint4*>(smem) + lane;
    // where a lane's rows of matrices begin: K, the next tile's in the upper half of the warp; V, the next piece's
    const uint32_t lane_k = Pieces<Shape::kRowK>::row_at(kTiles > 1 ? lane : lane & 15);
    using PiecesV = Pieces<Shape::kRowV>;
    const uint32_t lane_v = kUnit * Shape::kRowK + (PiecesV::kTurn > 0 ? PiecesV::at(PiecesV::row_at(lane & 15), lane >> 4)
                                                                       : PiecesV::row_at(lane & 15) + (lane >> 4) * 16);
    int turn = 0;
    for (int u = u0 + warp; u < u1; u += warps, ++turn) {
      const int stage = turn & 1;
      const uint32_t none = next_missing;
      cp_async_wait<0>();
      __syncwarp();
      next_missing = fetch(turn + 1, stage ^ 1);
      const uint32_t from_k = ring_at + stage * Shape::kStageBytes + lane_k, from_v = ring_at + stage * Shape::kStageBytes + lane_v;
      const uint8_t* const scales_k = ring + stage * Shape::kStageBytes + kUnit * (Shape::kRowK + Shape::kRowV);
      const uint8_t* const scales_v = scales_k + kUnit * Shape::kScaleK;

      // ---- S ----
      float s[kTiles][kN][4];
      if constexpr (kInt4) {
        uint32_t pairs[kTiles][2][kGroupsK];
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            load_words<kGroupsK>(pairs[i][half], reinterpret_cast<const uint32_t*>(scales_k) + (i * 16 + half * 8 + g) * kGroupsK);
#pragma unroll
        for (int group = 0; group < kGroupsK; ++group) {
          float acc[kTiles][kN][4] = {};
#pragma unroll
          for (int cc = 0; cc < Shape::kPerGroupK; ++cc) {
            const int c = group * Shape::kPerGroupK + cc;
            uint4 qf[kN];
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) qf[nb] = frags[(c * kN + nb) * 32];
            uint32_t words[kTiles][2];
            load_tiles<kTiles, Shape::kRowK>(Pieces<Shape::kRowK>::at(from_k, c), words);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              uint32_t w0 = words[i][0], w1 = words[i][1];  // rows g and g + 8: word t4 of the 16 bytes
              const uint32_t a[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
              w0 >>= 8;
              w1 >>= 8;
              const uint32_t a2[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
#pragma unroll
              for (int nb = 0; nb < kN; ++nb) {
                mma_f16(acc[i][nb], a, qf[nb].x, qf[nb].y);
                mma_f16(acc[i][nb], a2, qf[nb].z, qf[nb].w);
              }
            }
          }
          float2 sums[kN];
#pragma unroll
          for (int nb = 0; nb < kN; ++nb) sums[nb] = *reinterpret_cast<const float2*>(q_sums + group * kRows + nb * 8 + t4 * 2);
#pragma unroll
          for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t pair = pairs[i][j >> 1][group];
              const float zero = bf16_bits_to_float(pair), scale = __uint_as_float(pair & 0xffff0000u);
#pragma unroll
              for (int nb = 0; nb < kN; ++nb) {
                const float sum = j & 1 ? sums[nb].y : sums[nb].x;
                const float part = group == 0 ? zero * sum : fmaf(zero, sum, s[i][nb][j]);
                s[i][nb][j] = fmaf(scale, acc[i][nb][j], part);
              }
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int nb = 0; nb < kN; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][nb][j] = 0.f;
        uint4 qf[kN];
#pragma unroll
        for (int c = 0; c < Shape::kChunksK; ++c) {
          if (c % 2 == 0) {
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) qf[nb] = frags[(c / 2 * kN + nb) * 32];
          }
          uint32_t words[kTiles][2];
          load_tiles<kTiles, Shape::kRowK>(Pieces<Shape::kRowK>::at(from_k, c), words);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            const uint32_t w0 = words[i][0], w1 = words[i][1];
            const uint32_t a[4] = {e4m3x2_to_f16x2(w0), e4m3x2_to_f16x2(w1), e4m3x2_to_f16x2(w0 >> 16), e4m3x2_to_f16x2(w1 >> 16)};
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) mma_f16(s[i][nb], a, c % 2 == 0 ? qf[nb].x : qf[nb].z, c % 2 == 0 ? qf[nb].y : qf[nb].w);
          }
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float scale = bf16_bits_to_float(reinterpret_cast<const uint16_t*>(scales_k)[i * 16 + half * 8 + g]);
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) {
              s[i][nb][half * 2] *= scale;
              s[i][nb][half * 2 + 1] *= scale;
            }
          }
      }
      if (p.soft_cap > 0.f) {  // cap * tanh(x / cap) in units of log2
        const float inside = 1.f / p.soft_cap, outside = p.soft_cap * kLog2e;
#pragma unroll
        for (int nb = 0; nb < kN; ++nb) {
          const float2 f = *reinterpret_cast<const float2*>(factors + nb * 8 + t4 * 2);
#pragma unroll
          for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              const float2 t = tanh_each(make_float2(s[i][nb][j] * f.x * inside, s[i][nb][j + 1] * f.y * inside));
              s[i][nb][j] = t.x * outside;
              s[i][nb][j + 1] = t.y * outside;
            }
        }
      }

      // ---- what is seen ----
      const int token0 = keys.lo + u * kUnit;
      const bool whole = none == 0 && u >= whole_lo && u < whole_hi;
      uint32_t seen = ~0u;  // a bit for each of s, where not whole: tile, block, element
      // Of a unit's tokens, what no row sees (behind the end, without a page, before every window) may be anything, never written
      // maybe: it must not have a say in when sums are rescaled either, or last bits would hang on it.
      auto some_row_sees = [&](int token) {
        const int at = token0 + token, position = position0 + query_of(n_rows - 1);
        return at < keys.hi && at <= position && (p.window < 0 || at >= position0 - p.window) && !(none >> (token >> 4) & 1);
      };
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int nb = 0; nb < kN; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int position = position0 + query_of(min(nb * 8 + t4 * 2 + (j & 1), n_rows - 1));
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              const int token = token0 + i * 16 + (j >> 1) * 8 + g;
              const bool held = !(none >> i & 1) && token < keys.hi;
              const bool keep = held && token <= position && (p.window < 0 || token >= position - p.window);
              if (keep)
                seen |= 1u << ((i * kN + nb) * 4 + j);
              else
                s[i][nb][j] = -INFINITY;
            }
          }
      }
      static_assert(kTiles * kN * 4 <= 32);
      if (!kInt4 && !whole) {
        // V's codes of tokens that no row sees become 0: P is 0 there, but 0 times whatever lies there need not be.  (Codes of four
        // bits are numbers always.)
        constexpr int kEach = Shape::kRowV / 16;
        uint4* const values = reinterpret_cast<uint4*>(ring + stage * Shape::kStageBytes + kUnit * Shape::kRowK);
        for (int j = lane; j < kUnit * kEach; j += 32) {  // (a row's pieces are turned within the row)
          const int token = j / kEach;
          if (!some_row_sees(token)) values[j] = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }

      // ---- the maximum that P is taken against: raised where a logit passes its limit, kSlack above it ----
      constexpr int kLevel = kLevelTokens / kUnit;
      const bool level = kInt4 && turn % kLevel == kLevel - 1;
      bool grows = level;
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = fmaxf(s[0][nb][j], s[0][nb][2 + j]);
#pragma unroll
          for (int i = 1; i < kTiles; ++i) x = max3(x, s[i][nb][j], s[i][nb][2 + j]);
          const float most = x * factor[nb][j];
          highest[nb][j] = fmaxf(highest[nb][j], most);
          grows = grows || most > limit[nb][j];
        }
      // ---- and the power of two that P * scale is taken in: seen to where a scale passes `top` by a factor of two ----
      uint32_t own_top[(kUnit + 31) / 32][kGroupsV];  // a lane a token
#pragma unroll
      for (int i = 0; i < kUnit; i += 32) {
        const int token = kUnit < 32 ? lane & (kUnit - 1) : i + lane;
        if constexpr (kInt4)
          load_words<kGroupsV>(own_top[i / 32], reinterpret_cast<const uint32_t*>(scales_v) + token * kGroupsV);
        else
          own_top[i / 32][0] = (uint32_t)reinterpret_cast<const uint16_t*>(scales_v)[token] << 16;
        if (!whole && !some_row_sees(token)) {
#pragma unroll
          for (int group = 0; group < kGroupsV; ++group) own_top[i / 32][group] = 0;
        }
#pragma unroll
        for (int group = 0; group < kGroupsV; ++group) grows = grows || own_top[i / 32][group] >= top + (1u << 23);
      }
      if (__any_sync(~0u, grows)) {
        auto largest_of = [](const uint32_t (&scales)[kGroupsV]) {  // of a token, as bits (not NaN)
          uint32_t x = 0;
#pragma unroll
          for (int group = 0; group < kGroupsV; ++group) x = max(x, scales[group] < 0x7f800000u ? scales[group] : 0u);
          return x;
        };
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < kUnit; i += 32) {
          const uint32_t own = largest_of(own_top[i / 32]);
          largest = max(largest, own);
        }
        largest_seen = max(__reduce_max_sync(~0u, largest) & 0x7f800000u, largest_seen);
        const float largest_log2 = (float)((int)(largest_seen >> 23) - 127);
        float scale_log2[kTiles][2];  // of the tokens of s, rounded down
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int token = i * 16 + half * 8 + g;
            uint32_t own[kGroupsV];
            if constexpr (kInt4)
              load_words<kGroupsV>(own, reinterpret_cast<const uint32_t*>(scales_v) + token * kGroupsV);
            else
              own[0] = (uint32_t)reinterpret_cast<const uint16_t*>(scales_v)[token] << 16;
            scale_log2[i][half] = (float)((int)(largest_of(own) >> 23) - 127);
          }
        float least_log2 = largest_log2;
#pragma unroll
        for (int nb = 0; nb < kN; ++nb)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = highest[nb][j], w = -INFINITY;
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
              for (int half = 0; half < 2; ++half) w = fmaxf(w, fmaf(s[i][nb][half * 2 + j], factor[nb][j], scale_log2[i][half]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
              w = fmaxf(w, __shfl_xor_sync(~0u, w, d));
            }
            // of these keys, and of those before (whose unit `base` holds)
            float top_log2 = max3(w - x, base[nb][j] + kUnitLog2 - x, kLeastTopLog2);
            top_log2 = largest_log2 - top_log2 > kSpare ? top_log2 + kRoom : largest_log2;
            if (x > kNoMaximum) least_log2 = fminf(least_log2, top_log2);
            const float taken = x - kUnitLog2 + top_log2, alpha = ex2(base[nb][j] - taken);
            // Logits of 2^20 and more are 2^-3 apart and more, from 2^26 on as far as kSlack: no room between one and the next.  (`base`
            // is rounded as they are, and with it what P is taken in: up to some 2^27 f16 has room for that.  P from logits rounded
            // as the maximum is, which goes further, costs 1 to 3 %.)
            limit[nb][j] = fabsf(x) < 0x1p20f ? x + kSlack : x;
            base[nb][j] = taken;
            l[nb][j] *= alpha;
#pragma unroll
            for (int c = 0; c < Shape::kChunksV; ++c)
#pragma unroll
              for (int k = 0; k < kSteps; ++k) {
                o[c][k][nb][j] *= alpha;
                o[c][k][nb][2 + j] *= alpha;
              }
#pragma unroll
            for (int c = 0; c < kGroupsV; ++c) zeros[c][nb][j] *= alpha;
          }
        // The mean of a group's sums goes to its zeros from time to time: products of codes are positive, and a sum that MMAs add
        // up loses the bits that it cuts off at every step.
        if (level) {
#pragma unroll
          for (int group = 0; group < kGroupsV; ++group)
#pragma unroll
            for (int nb = 0; nb < kN; ++nb)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                constexpr int kPer = Shape::kPerGroupV;
                const float odd = p.dtype == SPLASH_F16 ? 1.f : 16.f, unit = p.dtype == SPLASH_F16 ? 1.f : kCodeUnit;
                float mean = 0.f;
#pragma unroll
                for (int c = group * kPer; c < (group + 1) * kPer; ++c)
#pragma unroll
                  for (int k = 0; k < kSteps; ++k) mean += fmaf(o[c][k][nb][2 + j], 1.f / odd, o[c][k][nb][j]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mean += __shfl_xor_sync(~0u, mean, d);
                mean *= 1.f / (kPer * 32);
#pragma unroll
                for (int c = group * kPer; c < (group + 1) * kPer; ++c)
#pragma unroll
                  for (int k = 0; k < kSteps; ++k) {
                    o[c][k][nb][j] -= mean;
                    o[c][k][nb][2 + j] = fmaf(-odd, mean, o[c][k][nb][2 + j]);
                  }
                zeros[group][nb][j] = fmaf(mean, unit / 8.f, zeros[group][nb][j]);  // (eight lanes')
              }
        }
        top = (uint32_t)(__reduce_min_sync(~0u, (int)floorf(least_log2)) + 127) << 23;
      }
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            s[i][nb][j] = ex2(fmaf(s[i][nb][j], factor[nb][j & 1], -base[nb][j & 1]));
            l[nb][j & 1] += s[i][nb][j];
          }

      // ---- O ----
      auto accumulate = [&](auto masked, auto fine) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          uint32_t pairs[2][kGroupsV], words[4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int token = i * 16 + half * 8 + g;
            if constexpr (kInt4)
              load_words<kGroupsV>(pairs[half], reinterpret_cast<const uint32_t*>(scales_v) + token * kGroupsV);
            else
              pairs[half][0] = (uint32_t)reinterpret_cast<const uint16_t*>(scales_v)[token] << 16;
          }
#pragma unroll
          for (int group = 0; group < kGroupsV; ++group) {
            uint32_t pf[kN][2];  // P * scale as the MMAs' second operand
            uint32_t rest[kN][2];  // fine: what that leaves of it
            float scale[2], zero[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              scale[half] = __uint_as_float(pairs[half][group] & 0xffff0000u);
              zero[half] = bf16_bits_to_float(pairs[half][group]);
              if (decltype(fine)::value) zero[half] = fmaf(scale[half], 8.f, zero[half]);  // of codes less 8
            }
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) {
              float x[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const bool dead = decltype(masked)::value && !(seen >> ((i * kN + nb) * 4 + j) & 1);
                x[j] = dead ? 0.f : s[i][nb][j] * scale[j >> 1];  // (whatever lies there, NaN too)
                if (kInt4 && !dead) zeros[group][nb][j & 1] = fmaf(s[i][nb][j], zero[j >> 1], zeros[group][nb][j & 1]);
              }
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const uint32_t pair = pack_f16(x[half * 2], x[half * 2 + 1]);
                pf[nb][half] = movmatrix(pair);
                if (decltype(fine)::value) {
                  const float2 kept = __half22float2(*reinterpret_cast<const __half2*>(&pair));
                  rest[nb][half] = movmatrix(pack_f16(x[half * 2] - kept.x, x[half * 2 + 1] - kept.y));
                }
              }
            }
#pragma unroll
            for (int cc = 0; cc < Shape::kPerGroupV; ++cc) {
              const int c = group * Shape::kPerGroupV + cc;
              // tokens 2 * t4 and the next (w1: + 8), 16 bits each from byte 2 * g of the piece; two pieces at a time
              if (c % 2 == 0) {
                const uint32_t at = Pieces<Shape::kRowV>::at(from_v, c) + i * 16 * Shape::kRowV;
                if (c + 1 < Shape::kChunksV)
                  ldmatrix_x4_trans(at, words[0], words[1], words[2], words[3]);
                else
                  ldmatrix_x2_trans(at, words[0], words[1]);
              }
              uint32_t w0 = words[c % 2 * 2], w1 = words[c % 2 * 2 + 1];
              if constexpr (kInt4) {
                auto codes = [](uint32_t word, bool odd) {
                  if (decltype(fine)::value) return less_eight(word, odd);
                  return word & (odd ? 0x00f000f0u : 0x000f000fu);
                };
                const uint32_t a[4] = {codes(w0, false), codes(w0, true), codes(w1, false), codes(w1, true)};
                w0 >>= 8;
                w1 >>= 8;
                const uint32_t a2[4] = {codes(w0, false), codes(w0, true), codes(w1, false), codes(w1, true)};
#pragma unroll
                for (int nb = 0; nb < kN; ++nb) {
                  mma_f16(o[c][0][nb], a, pf[nb][0], pf[nb][1]);
                  mma_f16(o[c][1][nb], a2, pf[nb][0], pf[nb][1]);
                  if (decltype(fine)::value) {
                    mma_f16(o[c][0][nb], a, rest[nb][0], rest[nb][1]);
                    mma_f16(o[c][1][nb], a2, rest[nb][0], rest[nb][1]);
                  }
                }
              } else {
                const uint32_t x0 = __byte_perm(w0, 0, 0x3120), x1 = __byte_perm(w1, 0, 0x3120);
                const uint32_t a[4] = {e4m3x2_to_f16x2(x0), e4m3x2_to_f16x2(x0 >> 16), e4m3x2_to_f16x2(x1), e4m3x2_to_f16x2(x1 >> 16)};
#pragma unroll
                for (int nb = 0; nb < kN; ++nb) {
                  mma_f16(o[c][0][nb], a, pf[nb][0], pf[nb][1]);
                  if (decltype(fine)::value) mma_f16(o[c][0][nb], a, rest[nb][0], rest[nb][1]);
                }
              }
            }
          }
        }
      };
      if (p.dtype == SPLASH_F16) {
        if (whole)
          accumulate(std::false_type{}, std::true_type{});
        else
          accumulate(std::true_type{}, std::true_type{});
      } else if (whole) {
        accumulate(std::false_type{}, std::false_type{});
      } else {
        accumulate(std::true_type{}, std::false_type{});
      }
      __syncwarp();
    }
    cp_async_wait<0>();  // (nothing is in flight that anyone waits for; the place of the stages is about to be written)
    __syncwarp();

    // ---- the sums of the warps that had units, each in its own place ----
    const int active = min(warps, u1 - u0);
    if (warp < active) {
      float* const own = reinterpret_cast<float*>(ring);
      // of products of int4 codes
      const float back = p.dtype == SPLASH_F16 ? 1.f : kCodeUnit, back_odd = p.dtype == SPLASH_F16 ? 1.f : kCodeUnit / 16.f;
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = nb * 8 + t4 * 2 + j;
          float sum = l[nb][j], high = highest[nb][j], z[kGroupsV];
#pragma unroll
          for (int c = 0; c < kGroupsV; ++c) z[c] = zeros[c][nb][j];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            sum += __shfl_xor_sync(~0u, sum, d);
            high = fmaxf(high, __shfl_xor_sync(~0u, high, d));
            if (kInt4) {
#pragma unroll
              for (int c = 0; c < kGroupsV; ++c) z[c] += __shfl_xor_sync(~0u, z[c], d);
            }
          }
          if (g == 0) {
            warp_high[warp * kRows + r] = high;
            warp_base[warp * kRows + r] = base[nb][j];
            warp_sum[warp * kRows + r] = sum;
          }
#pragma unroll
          for (int c = 0; c < Shape::kChunksV; ++c) {
            if constexpr (kInt4) {
              const float zero = z[c / Shape::kPerGroupV];
              *reinterpret_cast<float4*>(own + r * Shape::kV + c * 32 + g * 4) =
                  make_float4(fmaf(o[c][0][nb][j], back, zero), fmaf(o[c][0][nb][2 + j], back_odd, zero),
                              fmaf(o[c][1][nb][j], back, zero), fmaf(o[c][1][nb][2 + j], back_odd, zero));
            } else {
              *reinterpret_cast<float2*>(own + r * Shape::kV + c * 16 + g * 2) = make_float2(o[c][0][nb][j], o[c][0][nb][2 + j]);
            }
          }
        }
    }
    __syncthreads();
    // ---- and together ----
    if (clustered) cluster_wait();  // (the others are there)
    const bool alone = u0 == 0 && u1 == keys.units;
    // sums of this CTA: an item that began before its share in place 0, one that goes on behind it in place 1 (both: 0)
    float* const part = p.parts + ((int64_t)blockIdx.x * 2 + (is_last ? 1 : 0)) * (kRows * (Shape::kV + 2));
    for (int id = tid; id < n_rows * (Shape::kV / 8); id += blockDim.x) {
      const int r = id / (Shape::kV / 8), d = id % (Shape::kV / 8) * 8;
      float x[8] = {};
      float most = kNoMaximum, sum = 0.f;
      for (int w = 0; w < active; ++w) most = fmaxf(most, warp_high[w * kRows + r]);
#pragma unroll 4
      for (int w = 0; w < active; ++w) {
        const float weight = ex2(warp_base[w * kRows + r] - most);
        const uint8_t* const sums = smem + Shape::kRing + w * Shape::kWarpBytes;
        const float4* const from = reinterpret_cast<const float4*>(sums + (r * Shape::kV + d) * 4);
        const float4 lo = from[0], hi = from[1];
        const float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = fmaf(y[k], weight, x[k]);
        sum = fmaf(warp_sum[w * kRows + r], weight, sum);
      }
      if (clustered) {  // to the CTA that finishes these channels
        const uint32_t to = cluster_addr(received + (id / p.cluster * p.cluster + rank) * 12, id % p.cluster);
        cluster_st_v4(to, x[0], x[1], x[2], x[3]);
        cluster_st_v4(to + 16, x[4], x[5], x[6], x[7]);
        cluster_st_v4(to + 32, most, sum, 0.f, 0.f);
        continue;
      }
      if (!alone) {
        float4* const to = reinterpret_cast<float4*>(part + r * Shape::kV + d);
        to[0] = make_float4(x[0], x[1], x[2], x[3]);
        to[1] = make_float4(x[4], x[5], x[6], x[7]);
        if (d == 0) {
          part[kRows * Shape::kV + r] = most;
          part[kRows * (Shape::kV + 1) + r] = sum;
        }
        continue;
      }
      finish_row<kByHead>(p, rows, row0 + r, d, x, most, sum);
    }
    if (clustered) {  // (a cluster has one item)
      cluster_sync();
      for (int id = tid * p.cluster + rank; id < n_rows * (Shape::kV / 8); id += blockDim.x * p.cluster) {
        const float* const from = received + id / p.cluster * p.cluster * 12;
        float x[8] = {}, sum = 0.f, most = kNoMaximum;
        for (int c = 0; c < p.cluster; ++c) most = fmaxf(most, from[c * 12 + 8]);
#pragma unroll 4
        for (int c = 0; c < p.cluster; ++c) {
          const float weight = ex2(from[c * 12 + 8] - most);
          const float4 lo = *reinterpret_cast<const float4*>(from + c * 12), hi = *reinterpret_cast<const float4*>(from + c * 12 + 4);
          const float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = fmaf(y[k], weight, x[k]);
          sum = fmaf(from[c * 12 + 9], weight, sum);
        }
        finish_row<kByHead>(p, rows, row0 + id / (Shape::kV / 8), id % (Shape::kV / 8) * 8, x, most, sum);
      }
      return;
    }
    __syncthreads();  // before q's place, the statistics and the ring are written again
  }
}

// ------------------------------------------------------------------------------------------
// items that several CTAs have worked on, and items without keys
// ------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 256;

// blockIdx.x: row tile of an item (fastest) and head; y: sequence.  A thread has eight channels of a row; a row's parts are
// dealt to as many threads as there are parts for, so that a block takes several rows at a time where they are few.  z: the
// rows that a block takes are every gridDim.z-th such lot.
// kAhead: parts whose loads a thread has in flight together, which registers have to hold: four where there are few items, of
// many parts each, two and twice the blocks on an SM otherwise (us of a whole call, four : two; 8 items of 74 parts 41.3 : 42.7, 24
// items of some 25 20.7 : 21.6; 128 items of some 5 37.2 : 34.0, 512 of one or two 50.7 : 48.5).
template <int kRows, int kV, int kAhead, bool kByHead>
__global__ void __launch_bounds__(kJoinThreads, kAhead > 2 ? 2 : 4) cache_attend_join_kernel(const __grid_constant__ AttendParams p, int ctas) {
  constexpr int kEach = kV / 8, kLanes = kJoinThreads / kEach;  // threads of a row's channels; how many such lots
  constexpr int kMostSlices = kLanes >= 16 ? 16 : 8;
  static_assert(kLanes >= 8);
  constexpr int kPart = kRows * (kV + 2);
  __shared__ float sums[kMostSlices][kV];
  __shared__ float stats[2][kMostSlices];
  grid_dependency_wait();
  const int lot = threadIdx.x / kEach, d = threadIdx.x % kEach * 8;
  const int64_t share = share_of(p.starts[p.batch], ctas);
  for (int b = blockIdx.y; b < p.batch; b += gridDim.y) {
    const int64_t before = p.starts[b], cost = quotient(p.starts[b + 1] - before, items_of_table<kByHead>(p));
    const int64_t first = before + blockIdx.x * cost + p.item_cost;  // unit of this item
    const int64_t c0 = quotient(first, share), c1 = cost > 0 ? quotient(first + cost - p.item_cost - 1, share) : c0 - 1;
    if (c0 == c1) continue;  // written already
    const Rows rows = rows_of<kByHead>(p, b, blockIdx.x);
    const int row0 = blockIdx.x % p.row_tiles * kRows;
    const int n_rows = min(kRows, p.q_len * p.heads_per_kv - row0);
    int slices = 1;
    while (slices < kMostSlices && slices * 2 <= c1 - c0 + 1) slices *= 2;
    const int at_once = kMostSlices / slices, slice = lot % slices;
    for (int r0 = blockIdx.z * at_once; r0 < n_rows; r0 += gridDim.z * at_once) {
      const int r = r0 + lot / slices;
      float most = kNoMaximum, sum = 0.f, x[8] = {};
      const bool mine = lot < kMostSlices && r < n_rows;
      if (mine) {
        for (int64_t c = c0 + slice; c <= c1; c += slices * kAhead) {
          float m[kAhead], l[kAhead];
          float4 lo[kAhead], hi[kAhead];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const int64_t at = c + k * slices;
            m[k] = kNoMaximum;
            l[k] = 0.f;
            lo[k] = hi[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at > c1) continue;
            // the first CTA has the item last in its share, unless it starts there
            const float* const from = p.parts + at * (2 * kPart) + (at * share < first ? kPart : 0);
            m[k] = from[kRows * kV + r];
            l[k] = from[kRows * (kV + 1) + r];
            lo[k] = *reinterpret_cast<const float4*>(from + r * kV + d);
            hi[k] = *reinterpret_cast<const float4*>(from + r * kV + d + 4);
          }
          float top = most;
#pragma unroll
          for (int k = 0; k < kAhead; ++k) top = fmaxf(top, m[k]);
          const float old = ex2(most - top);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= old;
          sum *= old;
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const float weight = ex2(m[k] - top);
            const float y[8] = {lo[k].x, lo[k].y, lo[k].z, lo[k].w, hi[k].x, hi[k].y, hi[k].z, hi[k].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(y[i], weight, x[i]);
            sum = fmaf(l[k], weight, sum);
          }
          most = top;
        }
      }
      if (slices > 1) {  // (all threads of the block alike)
        if (mine && slice > 0) {
          *reinterpret_cast<float4*>(&sums[lot][d]) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(&sums[lot][d + 4]) = make_float4(x[4], x[5], x[6], x[7]);
          if (d == 0) {
            stats[0][lot] = most;
            stats[1][lot] = sum;
          }
        }
        __syncthreads();
        if (mine && slice == 0) {
          float top = most;
          for (int k = 1; k < slices; ++k) top = fmaxf(top, stats[0][lot + k]);
          const float own = ex2(most - top);
          sum *= own;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= own;
          for (int k = 1; k < slices; ++k) {
            const float weight = ex2(stats[0][lot + k] - top);
            sum = fmaf(stats[1][lot + k], weight, sum);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(sums[lot + k][d + i], weight, x[i]);
          }
          most = top;
        }
        __syncthreads();
      }
      if (mine && slice == 0) finish_row<kByHead>(p, rows, row0 + r, d, x, most, sum);
    }
  }
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
template <typename Shape, bool kByHead>
static int launch(const AttendParams& p, int warps, int ctas, cudaStream_t stream) {
  auto kernel = cache_attend_kernel<Shape, kByHead>;
  constexpr int kMostShared = kByHead ? Shape::smem_cluster(kMostWarps) : Shape::smem(kMostWarps);
  static_assert(kMostShared <= 227 * 1024);
  static std::atomic<uint64_t> ready{0};  // devices that know how much shared memory the kernel takes
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return SPLASH_ERR_CUDA;
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return SPLASH_ERR_CUDA;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t items = (int64_t)p.items * p.batch;
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attributes[2]{early_launch(), cluster_size(p.cluster)};
  config.attrs = attributes;
  config.stream = stream;
  // (shares: as many CTAs as the GPU holds; clusters: as many as there are items, which one alone takes in turn)
  config.gridDim = dim3((unsigned)(!p.whole ? ctas : p.cluster > 1 ? p.cluster * items : items < ctas ? items : ctas));
  config.blockDim = dim3(warps * 32);
  config.dynamicSmemBytes = p.cluster > 1 ? Shape::smem_cluster(warps) : Shape::smem(warps);
  config.numAttrs = kByHead ? p.cluster > 1 ? 2 : 1 : 0;
  if (cudaLaunchKernelEx(&config, kernel, p) != cudaSuccess) return SPLASH_ERR_CUDA;
  if (p.whole) return SPLASH_OK;
  config.dynamicSmemBytes = 0;
  config.numAttrs = 1;
  // (as many blocks of an item as its rows and the GPU have room for, where items are few)
  const int rows = p.q_len * p.heads_per_kv < Shape::kRows ? p.q_len * p.heads_per_kv : Shape::kRows;
  const bool few = items < kSms / 2;
  config.gridDim = dim3((unsigned)p.items, (unsigned)(p.batch < 65535 ? p.batch : 65535),
                        (unsigned)(items >= 2 * kSms ? 1 : items * rows <= 8 * kSms ? rows : 8 * kSms / items));
  config.blockDim = dim3(kJoinThreads);
  const auto join = few ? cache_attend_join_kernel<Shape::kRows, Shape::kV, 4, kByHead> : cache_attend_join_kernel<Shape::kRows, Shape::kV, 2, kByHead>;
  const cudaError_t launched = cudaLaunchKernelEx(&config, join, p, ctas);
  return launched == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

// CTAs that the GPU holds at a time
template <typename Shape>
constexpr int resident() {
  return kSms * Shape::kResident;
}

// Tokens of a sequence that the page table and the window let queries see.
static int64_t reach_of(const SplashCacheAttendArgs& a) {
  const int64_t reach = (int64_t)a.n_table * a.cache.page_size;
  return a.window >= 0 && reach > a.window + a.q.size[2] ? a.window + a.q.size[2] : reach;
}

constexpr int64_t kWideTokens = 1 << 18;

// Calls fn with the shape that a call takes.
template <typename Fn>
static int with_shape(const SplashCacheAttendArgs& a, Fn&& fn) {
  using std::integral_constant;
  const SplashKvCache& c = a.cache;
  const int64_t rows = a.q.size[2] * (a.q.size[1] / c.kv_heads);
  auto pick = [&](auto format, auto k, auto v, auto group) {
    constexpr int kF = decltype(format)::value, kK = decltype(k)::value, kV = decltype(v)::value, kG = decltype(group)::value;
    // Rows go in tiles of up to 16: the codes are read and unpacked again for each tile, but sums of more rows leave an SM
    // fewer warps.  Two exceptions, us measured:
    //   17 .. 24 rows of up to 128 channels are one tile (16 sequences of 2048 .. 4096 tokens, 32 / 8 heads of 128, 20 rows,
    //   int4 48.7 : 52.7, e4m3 44.6 : 49.1 in two tiles of 16; 32 rows in one tile 62.7, in two 55.0);
    //   rows of over 128 channels go by eight in small calls (one tile of 16 rows against two of 8, head dim 256: 32 x 8000 ..
    //   30000 tokens, 2 kv heads 122 : 139; 16 x 2000 .. 8000, 4 kv heads 55.1 : 55.4; 12 x 0 .. 10000, 1 kv head 23.2 : 20.8),
    //   below kWideTokens tokens times kv heads that the page tables have room for.
    if constexpr (kV <= 128) {
      if (rows > 16 && rows <= 24) return fn(AttendShape<kF, kK, kV, kG, 3>{});
    }
    const bool by_eight = rows <= 8 || (kV > 128 && reach_of(a) < kWideTokens / (a.q.size[0] * c.kv_heads));
    return by_eight ? fn(AttendShape<kF, kK, kV, kG, 1>{}) : fn(AttendShape<kF, kK, kV, kG, 2>{});
  };
  auto wide = [&](auto k, auto v) {
    constexpr int kK = decltype(k)::value, kV = decltype(v)::value;
    if (c.format == SPLASH_CACHE_E4M3) return pick(integral_constant<int, SPLASH_CACHE_E4M3>{}, k, v, integral_constant<int, 32>{});
    constexpr integral_constant<int, SPLASH_CACHE_INT4> int4;
    if constexpr (kK % 128 == 0 && kV % 128 == 0) {
      if (c.group == 128) return pick(int4, k, v, integral_constant<int, 128>{});
    }
    if constexpr (kK % 64 == 0 && kV % 64 == 0) {
      if (c.group == 64) return pick(int4, k, v, integral_constant<int, 64>{});
    }
    return pick(int4, k, v, integral_constant<int, 32>{});
  };
  switch (c.row_k) {
    case 64: return wide(integral_constant<int, 64>{}, integral_constant<int, 64>{});
    case 96: return wide(integral_constant<int, 96>{}, integral_constant<int, 96>{});
    case 128: return wide(integral_constant<int, 128>{}, integral_constant<int, 128>{});
    case 192:
      return c.row_v == 128 ? wide(integral_constant<int, 192>{}, integral_constant<int, 128>{})
                            : wide(integral_constant<int, 192>{}, integral_constant<int, 192>{});
    default: return wide(integral_constant<int, 256>{}, integral_constant<int, 256>{});
  }
}

// The sizes of a call with a table for each kv head and query: as many sequences of one query and one kv head.
static SplashCacheAttendArgs sizes_by_head(const SplashCacheAttendArgs& a) {
  SplashCacheAttendArgs s = a;
  for (SplashTensor* t : {&s.q, &s.o}) {
    t->size[0] *= a.cache.kv_heads * a.q.size[2];
    t->size[1] /= a.cache.kv_heads;
    t->size[2] = 1;
  }
  s.cache.kv_heads = 1;
  return s;
}

static int check_attend(const SplashCacheAttendArgs& a, bool by_head) {
  const SplashKvCache& c = a.cache;
  if (const int status = check_cache(c)) return status;
  for (const SplashTensor* t : {&a.q, &a.o})
    if (const int status = check_cache_tensor(*t, false)) return status;
  if (a.q.dtype != a.o.dtype) return SPLASH_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (a.q.size[i] != a.o.size[i]) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.q.size[3] != c.head_dim || a.o.size[3] != c.head_dim_v || a.q.size[1] % c.kv_heads != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.page_table == nullptr || a.lengths == nullptr || a.n_table <= 0 || a.table_stride < 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (!(a.soft_cap >= 0.f) || a.scale != a.scale) return SPLASH_ERR_INVALID_ARGUMENT;  // (not NaN)
  if (a.q.size[0] > (1 << 24) || a.q.size[1] > (1 << 20) || a.q.size[2] > (1 << 20) || a.q.size[1] * a.q.size[2] > (1 << 26) ||
      (int64_t)a.n_table * c.page_size > (1 << 30) ||
      c.n_pages * c.kv_heads > 0x7fffffffll / (c.page_size / 16))  // (tiles of 16 tokens are counted in 32 bits)
    return SPLASH_ERR_TOO_LARGE;
  if (by_head && a.window >= 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (by_head && a.q.size[0] * c.kv_heads * a.q.size[2] > (1 << 24)) return SPLASH_ERR_TOO_LARGE;
  return SPLASH_OK;
}

template <typename Shape>
static int64_t items_of(const SplashCacheAttendArgs& a) {
  const int64_t tiles = (a.q.size[2] * (a.q.size[1] / a.cache.kv_heads) + Shape::kRows - 1) / Shape::kRows;
  return a.q.size[0] * a.cache.kv_heads * tiles;
}

// Tables by head are of much the same length (so many pages of long sequences): an item can be one cluster's, of 1, 2, 4 or 8 CTAs of
// 4 or 8 warps, without shares to look for and a second launch.  What a call takes is estimated for each such form, in tokens of one
// SM with all its warps (265 a us, eight rows of 128 channels in int4: measured there alone, other shapes go by it too), and the least one taken:
//   * an SM has ceil(CTAs / SMs) of an item's parts, as many at a time as it holds; with 4, 8 and 12 warps it gets to 0.57, 0.92 and 0.97
//     of its rate, and another turn costs 4 us more (8 where it is clusters', which need room for all of their CTAs);
//   * a cluster's barriers and sums 0.35 us for each doubling; a warp has a unit at least;
//   * shares: equal for all SMs, and 4 us for the second launch and the search, 1.2 for each item of an SM.
// us measured, shares | 1 CTA of 8 warps | the form taken: 8 items of 1024 tokens 11.6 | 9.6 | 7.3 (8 x 8), of 8192 13.6 | 42.6 | 11.4 (8 x 8);
// 32 of 4096 14.8 | 23.8 | 11.3 (4 x 8), 192 of 4096 38.3 | 37.6 | 32.4 (2 x 4), 256 of 4096
// 45.7 | 37.6 | 37.6, 512 of 1024 23.1 | 27.0 | 23.1 (1 x 4).
struct Form {
  int cluster, warps;  // cluster 0: shares
};
template <typename Shape>
static Form form_by_head(const SplashCacheAttendArgs& a) {
  const double items = (double)items_of<Shape>(a), reach = (double)reach_of(a);
  Form best{0, kWarps};
  double least = 1100. + (1.05 * reach + 320.) * items / kSms;
  if (items > INT32_MAX / kMostCluster) return best;
  const auto rate = [](int warps) { return warps <= 4 ? 0.57 : warps <= 8 ? 0.92 : warps <= 12 ? 0.97 : 1.; };
  for (int cluster = 1, doublings = 0; cluster <= kMostCluster; cluster *= 2, ++doublings) {
    for (int warps = kWarps; warps <= kMostWarps; warps *= 2) {
      if (cluster > 1 && reach < (double)cluster * warps * Shape::kUnit) continue;
      const double held = std::max(Shape::kResident * kWarps / warps, 1), of_sm = std::ceil(items * cluster / kSms), part = reach / cluster;
      const double turns = std::floor(of_sm / held), rest = of_sm - turns * held;
      const double cost = turns * held * part / rate((int)held * warps) + (rest > 0. ? rest * part / rate((int)rest * warps) : 0.) +
                          (cluster > 1 ? 2200. : 1000.) * (std::ceil(of_sm / held) - 1.) + 100. * doublings;
      if (cost < least) least = cost, best = {cluster, warps};
    }
  }
  return best;
}

// Whether every item is given to one CTA: one launch, no sums in the workspace.
template <typename Shape>
static bool is_whole(const SplashCacheAttendArgs& a, bool by_head) {
  if (by_head) return form_by_head<Shape>(a).cluster > 0;
  const int64_t items = items_of<Shape>(a);
  const bool some = items >= kWholeItems && items < kMostWholeItems;
  return reach_of(a) <= (some ? 2 * kWholeTokens : kWholeTokens) && items <= INT32_MAX;
}

template <typename Shape>
static size_t parts_bytes() {
  return (size_t)resident<Shape>() * 2 * Shape::kRows * (Shape::kV + 2) * 4;
}

template <bool kByHead>
static int cache_attend(const SplashCacheAttendArgs& args, cudaStream_t stream) {
  if (const int status = check_attend(args, kByHead)) return status;
  const SplashCacheAttendArgs a = kByHead ? sizes_by_head(args) : args;
  const SplashKvCache& c = args.cache;
  AttendParams p{};
  p.k_codes = static_cast<const uint8_t*>(c.k_codes);
  p.k_scales = static_cast<const uint8_t*>(c.k_scales);
  p.v_codes = static_cast<const uint8_t*>(c.v_codes);
  p.v_scales = static_cast<const uint8_t*>(c.v_scales);
  p.q = a.q.data;
  p.o = a.o.data;
  p.page_table = a.page_table;
  p.lengths = a.lengths;
  p.lse = a.logsumexp;
  p.max_logits = a.max_logits;
  p.sinks = a.sinks;
  p.q_stride_b = a.q.stride[0], p.q_stride_h = a.q.stride[1], p.q_stride_s = a.q.stride[2];
  p.o_stride_b = a.o.stride[0], p.o_stride_h = a.o.stride[1], p.o_stride_s = a.o.stride[2];
  p.table_stride = a.table_stride;
  p.n_pages = c.n_pages;
  p.scale = a.scale;
  p.soft_cap = a.soft_cap;
  p.mask_value = a.mask_value;
  p.batch = (int32_t)a.q.size[0];
  p.q_heads = (int32_t)args.q.size[1];
  p.kv_heads = c.kv_heads;
  p.heads_per_kv = p.q_heads / c.kv_heads;
  p.q_len = (int32_t)a.q.size[2];
  p.queries = (int32_t)args.q.size[2];
  p.n_table = a.n_table;
  p.page_size = c.page_size;
  p.page_shift = log2_of(c.page_size);
  p.dtype = a.q.dtype;
  p.head_dim = c.head_dim;
  p.head_dim_v = c.head_dim_v;
  p.window = a.window < 0 ? -1 : a.window < (1 << 30) ? a.window : 1 << 30;  // (tables reach no further)
  return with_shape(a, [&](auto shape) -> int {
    using Shape = decltype(shape);
    AttendParams own = p;
    own.whole = is_whole<Shape>(a, kByHead);
    const int64_t items = items_of<Shape>(a);
    const Form form = kByHead ? form_by_head<Shape>(a) : Form{0, own.whole && items < 2 * kSms ? kMostWarps : kWarps};
    own.cluster = std::max(form.cluster, 1);
    if (!own.whole) {
      const size_t parts = parts_bytes<Shape>();
      if (a.workspace == nullptr || (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0 ||
          a.workspace_bytes < parts + 8 * ((size_t)p.batch + 1))
        return SPLASH_ERR_INVALID_ARGUMENT;
      own.parts = static_cast<float*>(a.workspace);
      own.starts = reinterpret_cast<int64_t*>(static_cast<uint8_t*>(a.workspace) + parts);
    }
    own.row_tiles = (p.q_len * p.heads_per_kv + Shape::kRows - 1) / Shape::kRows;
    own.items = a.cache.kv_heads * own.row_tiles;
    own.item_cost = item_tokens(Shape::kN) / Shape::kUnit;
    return launch<Shape, kByHead>(own, form.warps, resident<Shape>(), stream);
  });
}

static size_t cache_attend_workspace(const SplashCacheAttendArgs& args, bool by_head) {
  if (check_attend(args, by_head) != SPLASH_OK) return 0;
  const SplashCacheAttendArgs a = by_head ? sizes_by_head(args) : args;
  size_t bytes = 0;
  with_shape(a, [&](auto shape) -> int {
    using Shape = decltype(shape);
    if (!is_whole<Shape>(a, by_head)) bytes = parts_bytes<Shape>() + 8 * ((size_t)a.q.size[0] + 1);
    return 0;
  });
  return bytes;
}

}  // namespace sb
