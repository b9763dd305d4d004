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
//   * P * scale is scaled by a power of two that follows the largest scale seen (`top`), below 2^14: 11 bits of it are kept.
// Softmax statistics are of one pass over the keys, with a running maximum and sum for each row.
//
// Bound by: HBM, 64 + 8 bytes a token and head and side (int4, head dim 128, groups of 64); at 6.5 TB/s an SM gets 46 codes
// a cycle, so what counts beside the bytes in flight is the number of instructions for a code.
//
// Split: the keys of all (sequence, kv head, row tile) items, one after the other in units of kUnit tokens, are cut into
// equal shares for the CTAs, wherever that falls in a sequence.  A share is found on the device from the lengths: the host
// never needs them, and the launch can be captured in a graph.  The warps of a CTA take the units of its share of an
// item in turn, each with a ring of its own in shared memory (cp.async; no barrier between warps while keys stream), and
// join their sums at the end of the item.  An item that more than one CTA has worked on is joined by a second kernel, from
// sums in the workspace, in the order of the CTAs: results do not depend on who comes first.
#include "cache_common.cuh"

namespace sb {

constexpr int kAttendWarps = 8;
constexpr int kAttendThreads = kAttendWarps * 32;

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
  int64_t* starts;  // [batch + 1] first unit of each sequence
  int64_t q_stride_b, q_stride_h, q_stride_s, o_stride_b, o_stride_h, o_stride_s, table_stride, n_pages;
  float scale, soft_cap, mask_value;
  int32_t batch, q_heads, kv_heads, heads_per_kv, q_len, row_tiles, n_table, page_size, page_shift, group, group_shift, dtype;
  int32_t head_dim, head_dim_v, window, min_share;
};

// ------------------------------------------------------------------------------------------
// instructions
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_zeros(uint32_t dst, const void* somewhere) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, 0;" ::"r"(dst), "l"(somewhere) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x2(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(addr) : "memory");
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
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------------------------------
// sizes
// ------------------------------------------------------------------------------------------
// kK, kV: padded widths of a row; kN: blocks of eight query rows
template <int kFormat_, int kK_, int kV_, int kN_>
struct AttendShape {
  static constexpr int kFormat = kFormat_, kK = kK_, kV = kV_, kN = kN_;
  static constexpr bool kInt4 = kFormat == SPLASH_CACHE_INT4;
  static constexpr int kRows = 8 * kN;
  static constexpr int kRowK = cache_row_bytes(kFormat, kK), kRowV = cache_row_bytes(kFormat, kV);
  // tokens of a unit: about 4 KB, which a warp has in flight for each stage
  static constexpr int kUnit = kRowK + kRowV <= 64 ? 64 : kRowK + kRowV <= 128 ? 32 : 16;
  static constexpr int kTiles = kUnit / 16;
  // channels that 16 bytes of codes hold, and MMA steps (16 channels) over them
  static constexpr int kChunk = kInt4 ? 32 : 16, kSteps = kChunk / 16;
  static constexpr int kChunksK = kK / kChunk, kChunksV = kV / kChunk;
  static constexpr int kScaleK = kInt4 ? 4 * (kK / 32) : 2, kScaleV = kInt4 ? 4 * (kV / 32) : 2;  // at most
  static constexpr int kStageBytes = kUnit * (kRowK + kRowV + kScaleK + kScaleV);
  static constexpr int kStages = 3;
  static constexpr int kGroupsK = kInt4 ? kK / 32 : 1, kGroupsV = kInt4 ? kV / 32 : 1;  // at most
  // shared memory
  static constexpr int kFragBytes = kK / 16 * kN * 256;            // q as fragments
  static constexpr int kQSums = kFragBytes;                        // [kGroupsK][kRows] sums of q over a group
  static constexpr int kFactors = kQSums + kGroupsK * kRows * 4;   // [kRows] what S is multiplied by
  static constexpr int kStats = kFactors + kRows * 4;              // [2][kAttendWarps][kRows] maxima and sums of the warps
  static constexpr int kZeros = kStats + 2 * kAttendWarps * kRows * 4;  // [kAttendWarps][kGroupsV][kRows]
  static constexpr int kRing = (kZeros + kAttendWarps * kGroupsV * kRows * 4 + 127) / 128 * 128;
  static constexpr int kRingBytes = kAttendWarps * kStages * kStageBytes;
  static constexpr int kJoinBytes = kAttendWarps * kRows * kV * 4;  // in the ring's place once it has run dry
  static constexpr int kSmem = kRing + (kRingBytes > kJoinBytes ? kRingBytes : kJoinBytes);
};

// Where in a stage 16-byte piece c of row r lies: so that eight consecutive rows' piece c are in eight different bank groups.
template <int kRowBytes>
__device__ __forceinline__ int piece_at(int r, int c) {
  constexpr int kPieces = kRowBytes / 16;
  const int turn = kPieces % 8 == 0 ? r & 7 : kPieces % 4 == 0 ? (r >> 1) & 3 : kPieces % 2 == 0 ? (r >> 2) & 1 : 0;
  return r * kRowBytes + ((c ^ turn) << 4);
}

// ------------------------------------------------------------------------------------------
// shares
// ------------------------------------------------------------------------------------------
struct Keys {  // of a sequence: tokens [lo, hi) in whole units from lo, which is a multiple of kUnit
  int lo, hi, units;
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

__host__ __device__ inline int64_t share_of(int64_t total, int ctas, int min_share) {
  const int64_t share = (total + ctas - 1) / ctas;
  return share > min_share ? share : min_share;
}

struct Start {  // where a CTA's share begins
  int64_t total, before;  // units of all sequences (for one head and row tile), and before sequence b
  int b;
};

// All threads; `scratch`: 2 * kAttendWarps + 3 words of shared memory of 8 bytes.
template <int kUnit>
__device__ Start find_start(const AttendParams& p, int64_t* scratch) {
  const int per_sequence = p.kv_heads * p.row_tiles;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t total = 0, mine = 0;  // mine: of the sequences that this thread counts when there is one round of them
  for (int b = tid; b < p.batch; b += kAttendThreads) total += (mine = keys_of<kUnit>(p, __ldg(p.lengths + b)).units);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
  if (lane == 0) scratch[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kAttendWarps; ++w) total += scratch[w];
  const int64_t share = share_of(total * per_sequence, gridDim.x, p.min_share);
  const int64_t at = (int64_t)blockIdx.x * share;
  const bool keep = blockIdx.x == 0;  // this CTA writes down where the sequences start
  int64_t* found = scratch + 2 * kAttendWarps;
  int64_t carry = 0;
  for (int base = 0; base < p.batch; base += kAttendThreads) {
    const int b = base + tid;
    if (base > 0 || p.batch > kAttendThreads) mine = b < p.batch ? keys_of<kUnit>(p, __ldg(p.lengths + b)).units : 0;
    if (b >= p.batch) mine = 0;
    int64_t sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t other = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += other;
    }
    __syncthreads();
    if (lane == 31) scratch[kAttendWarps + warp] = sum;
    __syncthreads();
    int64_t before = carry, round = 0;
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) {
      const int64_t s = scratch[kAttendWarps + w];
      before += w < warp ? s : 0;
      round += s;
    }
    before += sum - mine;
    if (b < p.batch) {
      if (keep) p.starts[b] = before;
      if (mine > 0 && at >= before * per_sequence && at < (before + mine) * per_sequence) {
        found[0] = b;
        found[1] = before;
      }
    }
    carry += round;
  }
  if (keep && tid == 0) p.starts[p.batch] = total;
  __syncthreads();
  return {total, found[1], (int)found[0]};
}

// ------------------------------------------------------------------------------------------
// the kernel
// ------------------------------------------------------------------------------------------
// What a row's sums become: the output row, or a part of it in the workspace.  `m` in units of log2, with the sink in it.
__device__ __forceinline__ void add_sink(float sink, float& m, float& l) {
  const float s = sink * kLog2e, top = fmaxf(m, s);
  l = l * (m > -INFINITY ? ex2(m - top) : 0.f) + ex2(s - top);
  m = top;
}

template <typename Shape>
__global__ void __launch_bounds__(kAttendThreads) cache_attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kN = Shape::kN, kRows = Shape::kRows, kUnit = Shape::kUnit, kTiles = Shape::kTiles, kSteps = Shape::kSteps;
  constexpr bool kInt4 = Shape::kInt4;
  extern __shared__ __align__(128) uint8_t smem[];
  float* const q_sums = reinterpret_cast<float*>(smem + Shape::kQSums);
  float* const factors = reinterpret_cast<float*>(smem + Shape::kFactors);
  float* const warp_max = reinterpret_cast<float*>(smem + Shape::kStats);
  float* const warp_sum = warp_max + kAttendWarps * kRows;
  float* const warp_zeros = reinterpret_cast<float*>(smem + Shape::kZeros);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  grid_dependents_launch();  // the joining kernel may come up beside this one; it waits for its end

  const Start start = find_start<kUnit>(p, reinterpret_cast<int64_t*>(smem));
  __syncthreads();  // (its scratch is about to be q's place)
  const int per_sequence = p.kv_heads * p.row_tiles;
  const int64_t all = start.total * per_sequence, share = share_of(all, gridDim.x, p.min_share);
  int64_t at = (int64_t)blockIdx.x * share;
  const int64_t end = min(at + share, all);
  const int64_t first_unit = at;
  int b = start.b;
  int64_t before = start.before * per_sequence;  // units before sequence b
  const uint32_t ring = smem_u32(smem + Shape::kRing) + warp * (Shape::kStages * Shape::kStageBytes);
  const int groups_k = kInt4 ? Shape::kK >> p.group_shift : 1, groups_v = kInt4 ? Shape::kV >> p.group_shift : 1;
  const int chunk_mask = kInt4 ? (p.group >> 5) - 1 : 0;  // chunks of a group, less one
  const int scale_bytes_k = kInt4 ? 4 * groups_k : 2, scale_bytes_v = kInt4 ? 4 * groups_v : 2;
  const int heads = p.heads_per_kv;

  while (at < end) {
    Keys keys = keys_of<kUnit>(p, __ldg(p.lengths + b));
    while (at >= before + (int64_t)keys.units * per_sequence) {  // (sequences without keys are passed over)
      before += (int64_t)keys.units * per_sequence;
      keys = keys_of<kUnit>(p, __ldg(p.lengths + ++b));
    }
    const int length = __ldg(p.lengths + b);
    const int item = (int)((at - before) / keys.units);  // of this sequence: head * row_tiles + row tile
    const int head = item / p.row_tiles, row0 = item % p.row_tiles * kRows;
    const int64_t item_first = before + (int64_t)item * keys.units;
    const int u0 = (int)(at - item_first), u1 = (int)min((int64_t)keys.units, end - item_first);
    const int n_rows = min(kRows, p.q_len * heads - row0);
    const int32_t* const table = p.page_table + b * p.table_stride;

    // ---- keys on their way: unit u of this item into a stage ----
    // A unit's pages are looked up one turn ahead (lane i has tile i's).
    int next_page = -1;
    auto look_up = [&](int u) {
      const int token = keys.lo + u * kUnit + lane * 16;
      next_page = u < u1 && lane < kTiles && token < keys.hi ? __ldg(table + (token >> p.page_shift)) : -1;
      if (next_page >= p.n_pages) next_page = -1;
    };
    // Returns a bit for each tile of the unit that has no page (its keys are not seen).
    auto fetch = [&](int u, int stage) -> uint32_t {
      uint32_t missing = 0;
      if (u < u1) {
        const uint32_t to = ring + stage * Shape::kStageBytes;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const int page = __shfl_sync(~0u, next_page, i);
          if (page < 0) {
            missing |= 1u << i;
            // P is 0 there, but 0 times what lay there before need not be (codes of four bits are numbers always)
            if (!kInt4) {
#pragma unroll
              for (int j = 0; j < Shape::kRowV / 32; ++j)
                cp_async16_zeros(to + kUnit * Shape::kRowK + i * 16 * Shape::kRowV + (j * 32 + lane) * 16, p.v_codes);
            }
            continue;
          }
          const int token = keys.lo + u * kUnit + i * 16;
          const int64_t row = ((int64_t)page * p.kv_heads + head) * p.page_size + (token & (p.page_size - 1));
          const uint8_t* const k = p.k_codes + row * Shape::kRowK;
          const uint8_t* const v = p.v_codes + row * Shape::kRowV;
#pragma unroll
          for (int j = 0; j < (Shape::kRowK + 31) / 32; ++j) {
            const int piece = j * 32 + lane;
            if (Shape::kRowK % 32 == 0 || piece < Shape::kRowK)
              cp_async16(to + piece_at<Shape::kRowK>(i * 16 + piece / (Shape::kRowK / 16), piece % (Shape::kRowK / 16)), k + piece * 16);
          }
#pragma unroll
          for (int j = 0; j < (Shape::kRowV + 31) / 32; ++j) {
            const int piece = j * 32 + lane;
            if (Shape::kRowV % 32 == 0 || piece < Shape::kRowV)
              cp_async16(to + kUnit * Shape::kRowK + piece_at<Shape::kRowV>(i * 16 + piece / (Shape::kRowV / 16), piece % (Shape::kRowV / 16)),
                         v + piece * 16);
          }
          const uint32_t scales = to + kUnit * (Shape::kRowK + Shape::kRowV);
          if (lane < scale_bytes_k) cp_async16(scales + i * 16 * scale_bytes_k + lane * 16, p.k_scales + row * scale_bytes_k + lane * 16);
          if (lane < scale_bytes_v)
            cp_async16(scales + kUnit * Shape::kScaleK + i * 16 * scale_bytes_v + lane * 16, p.v_scales + row * scale_bytes_v + lane * 16);
        }
      }
      cp_async_commit();
      look_up(u + kAttendWarps);
      return missing;
    };
    static_assert(Shape::kStages == 3);
    look_up(u0 + warp);
    uint32_t missing[3];
    missing[0] = fetch(u0 + warp, 0);
    missing[1] = fetch(u0 + warp + kAttendWarps, 1);

    // ---- q as fragments; a warp a row ----
    for (int r = warp; r < kRows; r += kAttendWarps) {
      float x[8] = {};
      if (r < n_rows && lane * 8 < p.head_dim) {
        const int row = row0 + r, i = row / heads, h = head * heads + row % heads;
        load8(p.q, p.dtype, b * p.q_stride_b + h * p.q_stride_h + i * p.q_stride_s + lane * 8, x);
      }
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      // the power of two that brings `top` to 2^14 .. 2^15, within 2^-100 .. 2^100
      const int e = min(max((int)(__float_as_uint(top) >> 23), 41), 227);
      const float up = __uint_as_float((uint32_t)(268 - e) << 23), down = __uint_as_float((uint32_t)(e - 14) << 23);
      uint16_t h16[8];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half h = __float2half_rn(x[i] * up);
        h16[i] = __half_as_ushort(h);
        sum += __half2float(h);
        // int4: the odd codes of a half-word stand four bits higher
        if (kInt4 && (i & 1)) h16[i] = __half_as_ushort(__float2half_rn(__half2float(h) * 0.0625f));
      }
      auto two = [&](int lo, int hi) { return (uint32_t)h16[lo] | (uint32_t)h16[hi] << 16; };
      if (lane * 8 < Shape::kK) {
        uint2* const frag = reinterpret_cast<uint2*>(smem);
        const int block = r >> 3, n = r & 7;
        if (kInt4) {  // a lane's eight channels are one word of codes: steps 2 * (lane / 4) and the next, column lane % 4
          frag[((lane >> 2) * 2 * kN + block) * 32 + n * 4 + (lane & 3)] = make_uint2(two(0, 4), two(1, 5));
          frag[(((lane >> 2) * 2 + 1) * kN + block) * 32 + n * 4 + (lane & 3)] = make_uint2(two(2, 6), two(3, 7));
        } else {  // two words of codes: columns 2 * (lane % 2) and the next of step lane / 2
          frag[((lane >> 1) * kN + block) * 32 + n * 4 + (lane & 1) * 2] = make_uint2(two(0, 1), two(2, 3));
          frag[((lane >> 1) * kN + block) * 32 + n * 4 + (lane & 1) * 2 + 1] = make_uint2(two(4, 5), two(6, 7));
        }
      }
      if (kInt4) {
        for (int d = 1; d < p.group / 8; d <<= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if ((lane & (p.group / 8 - 1)) == 0 && lane * 8 < Shape::kK)
          q_sums[(lane * 8 >> p.group_shift) * kRows + r] = sum * 0x1p-24f;  // in the units of the products of codes
      }
      if (lane == 0) factors[r] = p.scale * down * (kInt4 ? 0x1p24f : 1.f) * (p.soft_cap > 0.f ? 1.f : kLog2e);
    }
    __syncthreads();

    // ---- this lane's columns: rows nb * 8 + t4 * 2 and the next ----
    float m[kN][2], l[kN][2], factor[kN][2];
    int last[kN][2];  // position of the query
    float o[Shape::kChunksV][kSteps][kN][4] = {};
    float zeros[Shape::kGroupsV][kN][2] = {};
    uint32_t top = 20u << 23;  // the largest scale of V seen (as bits), rounded down to a power of two
    int last_least = INT32_MAX, last_most = INT32_MIN;
#pragma unroll
    for (int nb = 0; nb < kN; ++nb)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = nb * 8 + t4 * 2 + j;
        m[nb][j] = -INFINITY;
        l[nb][j] = 0.f;
        factor[nb][j] = factors[r];
        last[nb][j] = length - p.q_len + (row0 + min(r, n_rows - 1)) / heads;
      }
    last_least = length - p.q_len + row0 / heads;
    last_most = length - p.q_len + (row0 + n_rows - 1) / heads;

    const uint2* const frags = reinterpret_cast<const uint2*>(smem) + lane;
    int stage = 0;
    for (int u = u0 + warp; u < u1; u += kAttendWarps) {
      cp_async_wait<1>();
      __syncwarp();
      const uint32_t none = missing[0];
      missing[0] = missing[1];
      missing[1] = fetch(u + 2 * kAttendWarps, stage == 0 ? 2 : stage - 1);
      const uint32_t from = ring + stage * Shape::kStageBytes;
      const uint8_t* const scales_k = smem + (from - smem_u32(smem)) + kUnit * (Shape::kRowK + Shape::kRowV);
      const uint8_t* const scales_v = scales_k + kUnit * Shape::kScaleK;
      stage = stage == 2 ? 0 : stage + 1;

      // ---- S ----
      float s[kTiles][kN][4];
      float acc[kTiles][kN][4];
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int nb = 0; nb < kN; ++nb)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][nb][j] = acc[i][nb][j] = 0.f;
#pragma unroll
      for (int c = 0; c < Shape::kChunksK; ++c) {
        uint2 qf[kSteps][kN];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int nb = 0; nb < kN; ++nb) qf[k][nb] = frags[((c * kSteps + k) * kN + nb) * 32];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          uint32_t w0, w1;  // rows g and g + 8: word t4 of the 16 bytes
          ldmatrix_x2(from + piece_at<Shape::kRowK>(i * 16 + (lane & 15), c), w0, w1);
          if (kInt4) {
            const uint32_t a[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
            w0 >>= 8;
            w1 >>= 8;
            const uint32_t a2[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) {
              mma_f16(acc[i][nb], a, qf[0][nb].x, qf[0][nb].y);
              mma_f16(acc[i][nb], a2, qf[kSteps - 1][nb].x, qf[kSteps - 1][nb].y);
            }
          } else {
            const uint32_t a[4] = {e4m3x2_to_f16x2(w0), e4m3x2_to_f16x2(w1), e4m3x2_to_f16x2(w0 >> 16), e4m3x2_to_f16x2(w1 >> 16)};
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) mma_f16(acc[i][nb], a, qf[0][nb].x, qf[0][nb].y);
          }
        }
        if (kInt4 && (c & chunk_mask) == chunk_mask) {  // the end of a group
          const int group = (c * 32) >> p.group_shift;
          float2 sums[kN];
#pragma unroll
          for (int nb = 0; nb < kN; ++nb) sums[nb] = *reinterpret_cast<const float2*>(q_sums + group * kRows + nb * 8 + t4 * 2);
#pragma unroll
          for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t pair = reinterpret_cast<const uint32_t*>(scales_k)[(i * 16 + half * 8 + g) * groups_k + group];
              const float zero = bf16_bits_to_float(pair), scale = __uint_as_float(pair & 0xffff0000u);
#pragma unroll
              for (int nb = 0; nb < kN; ++nb) {
                s[i][nb][half * 2] = fmaf(zero, sums[nb].x, fmaf(scale, acc[i][nb][half * 2], s[i][nb][half * 2]));
                s[i][nb][half * 2 + 1] = fmaf(zero, sums[nb].y, fmaf(scale, acc[i][nb][half * 2 + 1], s[i][nb][half * 2 + 1]));
                acc[i][nb][half * 2] = acc[i][nb][half * 2 + 1] = 0.f;
              }
            }
        }
      }
      // logits in units of log2
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float scale = 1.f;
          if (!kInt4) scale = bf16_bits_to_float(reinterpret_cast<const uint16_t*>(scales_k)[i * 16 + half * 8 + g]);
#pragma unroll
          for (int nb = 0; nb < kN; ++nb)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& x = s[i][nb][half * 2 + j];
              x = kInt4 ? x * factor[nb][j] : acc[i][nb][half * 2 + j] * scale * factor[nb][j];
              if (p.soft_cap > 0.f) {  // cap * tanh(x / cap), tanh y = 1 - 2 / (exp(2 y) + 1)
                const float e = ex2(x * (2.f * kLog2e / p.soft_cap));
                x = (p.soft_cap * kLog2e) * (1.f - __fdividef(2.f, e + 1.f));
              }
            }
        }

      // ---- what is seen ----
      const int token0 = keys.lo + u * kUnit;
      const bool whole = none == 0 && token0 + kUnit - 1 <= min(last_least, keys.hi - 1) && (p.window < 0 || token0 >= last_most - p.window);
      uint32_t seen = ~0u;  // a bit for each of s, where not whole: tile, block, element
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int nb = 0; nb < kN; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int token = token0 + i * 16 + (j >> 1) * 8 + g, position = last[nb][j & 1];
              const bool keep = !(none >> i & 1) && token < keys.hi && token <= position && (p.window < 0 || token >= position - p.window);
              if (keep)
                seen |= 1u << ((i * kN + nb) * 4 + j);
              else
                s[i][nb][j] = -INFINITY;
            }
      }
      static_assert(kTiles * kN * 4 <= 32);

      // ---- running maximum, P ----
      float alpha[kN][2];
      bool grew = false;
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top_s = -INFINITY;
#pragma unroll
          for (int i = 0; i < kTiles; ++i) top_s = max3(top_s, s[i][nb][j], s[i][nb][2 + j]);
          top_s = fmaxf(top_s, __shfl_xor_sync(~0u, top_s, 4));
          top_s = fmaxf(top_s, __shfl_xor_sync(~0u, top_s, 8));
          top_s = fmaxf(top_s, __shfl_xor_sync(~0u, top_s, 16));
          const float next = fmaxf(m[nb][j], top_s);
          grew = grew || next > m[nb][j];
          alpha[nb][j] = m[nb][j] > -INFINITY ? ex2(m[nb][j] - next) : 0.f;
          m[nb][j] = next;
          const float base = next > -INFINITY ? next : 0.f;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float& x = s[i][nb][half * 2 + j];
              x = ex2(x - base);
              sum += x;
            }
          l[nb][j] = l[nb][j] * alpha[nb][j] + sum;
        }

      // ---- the power of two that P * scale is taken in ----
      uint32_t largest = 0;
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int token = i * 16 + half * 8 + g;
          // (lanes t4 = 0 .. 3 have the same token: each looks at a quarter of its groups)
          if (kInt4) {
            for (int group = t4; group < groups_v; group += 4) {
              const uint32_t pair = reinterpret_cast<const uint32_t*>(scales_v)[token * groups_v + group];
              if ((whole || (!(none >> i & 1) && token0 + token < keys.hi)) && pair < 0x7f800000u) largest = max(largest, pair);
            }
          } else {
            const uint32_t bits = (uint32_t)reinterpret_cast<const uint16_t*>(scales_v)[token] << 16;
            if ((whole || (!(none >> i & 1) && token0 + token < keys.hi)) && bits < 0x7f800000u) largest = max(largest, bits);
          }
        }
      largest = __reduce_max_sync(~0u, largest) & 0x7f800000u;
      float rise = 1.f;  // what sums so far are multiplied by when it changes
      if (largest > top) {
        rise = __uint_as_float((uint32_t)max(127 - (int)((largest - top) >> 23), 0) << 23);
        top = largest;
      }
      const float unit = __uint_as_float((267u << 23) - top);  // 2^13 / 2^exponent(top)
      if (__any_sync(~0u, grew) || rise != 1.f) {
#pragma unroll
        for (int nb = 0; nb < kN; ++nb)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float a = alpha[nb][j] * rise;
#pragma unroll
            for (int c = 0; c < Shape::kChunksV; ++c)
#pragma unroll
              for (int k = 0; k < kSteps; ++k) {
                o[c][k][nb][j] *= a;
                o[c][k][nb][2 + j] *= a;
              }
#pragma unroll
            for (int c = 0; c < Shape::kGroupsV; ++c) zeros[c][nb][j] *= alpha[nb][j];
          }
      }

      // ---- O ----
      const uint32_t from_v = from + kUnit * Shape::kRowK;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        uint32_t pf[kN][2];  // P * scale as the MMAs' second operand
#pragma unroll
        for (int c = 0; c < Shape::kChunksV; ++c) {
          if (kInt4 ? (c & chunk_mask) == 0 : c == 0) {  // the start of a group
            const int group = kInt4 ? (c * 32) >> p.group_shift : 0;
            float scale[2], zero[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int token = i * 16 + half * 8 + g;
              if (kInt4) {
                const uint32_t pair = reinterpret_cast<const uint32_t*>(scales_v)[token * groups_v + group];
                zero[half] = bf16_bits_to_float(pair);
                scale[half] = __uint_as_float(pair & 0xffff0000u) * unit;
              } else {
                scale[half] = bf16_bits_to_float(reinterpret_cast<const uint16_t*>(scales_v)[token]) * unit;
              }
            }
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) {
              float x[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                x[j] = s[i][nb][j] * scale[j >> 1];
                float z = kInt4 ? s[i][nb][j] * zero[j >> 1] : 0.f;
                if (!whole && !(seen >> ((i * kN + nb) * 4 + j) & 1)) x[j] = z = 0.f;  // (whatever lies there, NaN too)
                if (kInt4) zeros[c][nb][j & 1] += z;
              }
              pf[nb][0] = movmatrix(pack_f16(x[0], x[1]));
              pf[nb][1] = movmatrix(pack_f16(x[2], x[3]));
            }
          }
          uint32_t w0, w1;  // tokens 2 * t4 and the next (w1: + 8), 16 bits each from byte 2 * g of the piece
          ldmatrix_x2_trans(from_v + piece_at<Shape::kRowV>(i * 16 + (lane & 15), c), w0, w1);
          if (kInt4) {
            const uint32_t a[4] = {w0 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x000f000fu, w1 & 0x00f000f0u};
            w0 >>= 8;
            w1 >>= 8;
            const uint32_t a2[4] = {w0 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x000f000fu, w1 & 0x00f000f0u};
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) {
              mma_f16(o[c][0][nb], a, pf[nb][0], pf[nb][1]);
              mma_f16(o[c][kSteps - 1][nb], a2, pf[nb][0], pf[nb][1]);
            }
          } else {
            const uint32_t x0 = __byte_perm(w0, 0, 0x3120), x1 = __byte_perm(w1, 0, 0x3120);
            const uint32_t a[4] = {e4m3x2_to_f16x2(x0), e4m3x2_to_f16x2(x0 >> 16), e4m3x2_to_f16x2(x1), e4m3x2_to_f16x2(x1 >> 16)};
#pragma unroll
            for (int nb = 0; nb < kN; ++nb) mma_f16(o[c][0][nb], a, pf[nb][0], pf[nb][1]);
          }
        }
      }
      __syncwarp();
    }
    cp_async_wait<0>();  // (nothing is in flight here that anyone waits for; the ring's place is about to be written)

    // ---- the warps' sums together ----
#pragma unroll
    for (int nb = 0; nb < kN; ++nb)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[nb][j];
        sum += __shfl_xor_sync(~0u, sum, 4);
        sum += __shfl_xor_sync(~0u, sum, 8);
        sum += __shfl_xor_sync(~0u, sum, 16);
        l[nb][j] = sum;
        if (kInt4) {
#pragma unroll
          for (int c = 0; c < Shape::kGroupsV; ++c) {
            float z = zeros[c][nb][j];
            z += __shfl_xor_sync(~0u, z, 4);
            z += __shfl_xor_sync(~0u, z, 8);
            z += __shfl_xor_sync(~0u, z, 16);
            if (lane < 4) warp_zeros[(warp * Shape::kGroupsV + c) * kRows + nb * 8 + t4 * 2 + j] = z;
          }
        }
        if (lane < 4) {
          warp_max[warp * kRows + nb * 8 + t4 * 2 + j] = m[nb][j];
          warp_sum[warp * kRows + nb * 8 + t4 * 2 + j] = sum;
        }
      }
    __syncthreads();
    {
      float* const join = reinterpret_cast<float*>(smem + Shape::kRing) + warp * (kRows * Shape::kV);
      const float back = __uint_as_float(top - (13u << 23)) * (kInt4 ? 0x1p24f : 1.f);  // 1 / unit
#pragma unroll
      for (int nb = 0; nb < kN; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = nb * 8 + t4 * 2 + j;
          float most = -INFINITY;
#pragma unroll
          for (int w = 0; w < kAttendWarps; ++w) most = fmaxf(most, warp_max[w * kRows + r]);
          const float weight = m[nb][j] > -INFINITY ? ex2(m[nb][j] - most) : 0.f;
#pragma unroll
          for (int c = 0; c < Shape::kChunksV; ++c) {
            if (kInt4) {
              const float4 x = make_float4(o[c][0][nb][j] * back, o[c][0][nb][2 + j] * (back * 0.0625f),
                                           o[c][kSteps - 1][nb][j] * back, o[c][kSteps - 1][nb][2 + j] * (back * 0.0625f));
              const float z = warp_zeros[(warp * Shape::kGroupsV + (c & ~chunk_mask)) * kRows + r];
              *reinterpret_cast<float4*>(join + r * Shape::kV + c * 32 + g * 4) =
                  make_float4((x.x + z) * weight, (x.y + z) * weight, (x.z + z) * weight, (x.w + z) * weight);
            } else {
              *reinterpret_cast<float2*>(join + r * Shape::kV + c * 16 + g * 2) =
                  make_float2(o[c][0][nb][j] * back * weight, o[c][0][nb][2 + j] * back * weight);
            }
          }
        }
    }
    __syncthreads();
    const bool alone = u0 == 0 && u1 == keys.units;
    // sums of this CTA: its first item in place 0, its last in place 1 (an item that is both and not whole: 0)
    float* const part = p.parts + ((int64_t)blockIdx.x * 2 + (at == first_unit ? 0 : 1)) * (kRows * (Shape::kV + 2));
    for (int id = tid; id < n_rows * (Shape::kV / 8); id += kAttendThreads) {
      const int r = id / (Shape::kV / 8), d = id % (Shape::kV / 8) * 8;
      float x[8] = {};
      float most = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) most = fmaxf(most, warp_max[w * kRows + r]);
#pragma unroll
      for (int w = 0; w < kAttendWarps; ++w) {
        const float mine = warp_max[w * kRows + r];
        sum += mine > -INFINITY ? warp_sum[w * kRows + r] * ex2(mine - most) : 0.f;
        const float4* const from = reinterpret_cast<const float4*>(reinterpret_cast<float*>(smem + Shape::kRing) + (w * kRows + r) * Shape::kV + d);
        const float4 lo = from[0], hi = from[1];
        x[0] += lo.x, x[1] += lo.y, x[2] += lo.z, x[3] += lo.w, x[4] += hi.x, x[5] += hi.y, x[6] += hi.z, x[7] += hi.w;
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
      const int row = row0 + r, i = row / heads, h = head * heads + row % heads;
      if (p.sinks != nullptr) {
        const float own = most;
        add_sink(__ldg(p.sinks + h), most, sum);
        const float weight = own > -INFINITY ? ex2(own - most) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= weight;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = sum == 0.f ? 0.f : x[k] * inv;
      if (d < p.head_dim_v) store8(p.o, p.dtype, b * p.o_stride_b + h * p.o_stride_h + i * p.o_stride_s + d, x);
      if (d == 0) {
        const int64_t to = ((int64_t)b * p.q_heads + h) * p.q_len + i;
        if (p.lse != nullptr) p.lse[to] = sum == 0.f ? p.mask_value : (most + __log2f(sum)) * kLn2;
        if (p.max_logits != nullptr) p.max_logits[to] = sum == 0.f ? p.mask_value : most * kLn2;
      }
    }
    at = item_first + u1;
    __syncthreads();  // before q's place, the statistics and the ring are written again
  }
}

// ------------------------------------------------------------------------------------------
// items that several CTAs have worked on, and items without keys
// ------------------------------------------------------------------------------------------
constexpr int kJoinThreads = 128;

// blockIdx.x: row tile of an item (fastest) and head; y: sequence.  A thread has eight channels of a row.
template <int kRows, int kV>
__global__ void __launch_bounds__(kJoinThreads) cache_attend_join_kernel(const __grid_constant__ AttendParams p, int ctas) {
  grid_dependency_wait();
  const int per_sequence = p.kv_heads * p.row_tiles;
  for (int b = blockIdx.y; b < p.batch; b += gridDim.y) {
    const int64_t before = p.starts[b], units = p.starts[b + 1] - before;
    const int64_t share = share_of(p.starts[p.batch] * per_sequence, ctas, p.min_share);
    const int64_t first = before * per_sequence + blockIdx.x * units;  // unit of this item
    const int64_t c0 = first / share, c1 = units > 0 ? (first + units - 1) / share : c0 - 1;
    if (c0 == c1) continue;  // written already
    const int head = blockIdx.x / p.row_tiles, row0 = blockIdx.x % p.row_tiles * kRows;
    const int n_rows = min(kRows, p.q_len * p.heads_per_kv - row0);
    for (int id = threadIdx.x; id < n_rows * (kV / 8); id += kJoinThreads) {
      const int r = id / (kV / 8), d = id % (kV / 8) * 8;
      const int row = row0 + r, i = row / p.heads_per_kv, h = head * p.heads_per_kv + row % p.heads_per_kv;
      float most = -INFINITY, sum = 0.f, x[8] = {};
      for (int64_t c = c0; c <= c1; ++c) {
        // the first CTA has the item last in its share, unless it starts there
        const float* const part = p.parts + (c * 2 + (c * share < first ? 1 : 0)) * (kRows * (kV + 2));
        const float m = part[kRows * kV + r], l = part[kRows * (kV + 1) + r];
        const float4* const from = reinterpret_cast<const float4*>(part + r * kV + d);
        const float4 lo = from[0], hi = from[1];
        const float top = fmaxf(most, m);
        const float old = most > -INFINITY ? ex2(most - top) : 0.f, fresh = m > -INFINITY ? ex2(m - top) : 0.f;
        const float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = x[k] * old + y[k] * fresh;
        sum = sum * old + l * fresh;
        most = top;
      }
      if (p.sinks != nullptr) {
        const float own = most;
        add_sink(__ldg(p.sinks + h), most, sum);
        const float weight = own > -INFINITY ? ex2(own - most) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= weight;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = sum == 0.f ? 0.f : x[k] / sum;
      if (d < p.head_dim_v) store8(p.o, p.dtype, b * p.o_stride_b + h * p.o_stride_h + i * p.o_stride_s + d, x);
      if (d == 0) {
        const int64_t to = ((int64_t)b * p.q_heads + h) * p.q_len + i;
        if (p.lse != nullptr) p.lse[to] = sum == 0.f ? p.mask_value : (most + __log2f(sum)) * kLn2;
        if (p.max_logits != nullptr) p.max_logits[to] = sum == 0.f ? p.mask_value : most * kLn2;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
struct AttendPlan {
  int rows, ctas;
};

template <typename Shape>
static int launch(const AttendParams& p, int ctas, cudaStream_t stream) {
  auto kernel = cache_attend_kernel<Shape>;
  static_assert(Shape::kSmem <= 227 * 1024);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem) != cudaSuccess) return SPLASH_ERR_CUDA;
  kernel<<<ctas, kAttendThreads, Shape::kSmem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return SPLASH_ERR_CUDA;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(p.kv_heads * p.row_tiles), (unsigned)(p.batch < 65535 ? p.batch : 65535));
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, cache_attend_join_kernel<Shape::kRows, Shape::kV>, p, ctas) == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

// CTAs that the GPU holds at a time
template <typename Shape>
constexpr int resident() {
  return kSms * (Shape::kSmem <= 113 * 1024 ? 2 : 1);
}

// Calls fn with the shape that a call takes.
template <typename Fn>
static int with_shape(const SplashCacheAttendArgs& a, Fn&& fn) {
  const SplashKvCache& c = a.cache;
  const int64_t rows = a.q.size[2] * (a.q.size[1] / c.kv_heads);
  auto pick = [&](auto format) {
    constexpr int kF = decltype(format)::value;
    auto wide = [&](auto k, auto v) {
      constexpr int kK = decltype(k)::value, kV = decltype(v)::value;
      // eight rows a CTA, or sixteen, which unpack the codes once for twice as many
      if (rows <= 8 || kV > 128) return fn(AttendShape<kF, kK, kV, 1>{});
      return fn(AttendShape<kF, kK, kV, kV <= 128 ? 2 : 1>{});
    };
    using std::integral_constant;
    switch (c.row_k) {
      case 64: return wide(integral_constant<int, 64>{}, integral_constant<int, 64>{});
      case 96: return wide(integral_constant<int, 96>{}, integral_constant<int, 96>{});
      case 128: return wide(integral_constant<int, 128>{}, integral_constant<int, 128>{});
      case 192:
        return c.row_v == 128 ? wide(integral_constant<int, 192>{}, integral_constant<int, 128>{})
                              : wide(integral_constant<int, 192>{}, integral_constant<int, 192>{});
      default: return wide(integral_constant<int, 256>{}, integral_constant<int, 256>{});
    }
  };
  return c.format == SPLASH_CACHE_INT4 ? pick(std::integral_constant<int, SPLASH_CACHE_INT4>{})
                                       : pick(std::integral_constant<int, SPLASH_CACHE_E4M3>{});
}

static int check_attend(const SplashCacheAttendArgs& a) {
  const SplashKvCache& c = a.cache;
  if (const int status = check_cache(c)) return status;
  for (const SplashTensor* t : {&a.q, &a.o})
    if (const int status = check_cache_tensor(*t, false)) return status;
  if (a.q.dtype != a.o.dtype) return SPLASH_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (a.q.size[i] != a.o.size[i]) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.q.size[3] != c.head_dim || a.o.size[3] != c.head_dim_v || a.q.size[1] % c.kv_heads != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.page_table == nullptr || a.lengths == nullptr || a.n_table <= 0 || a.table_stride < 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (!(a.soft_cap >= 0.f)) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.q.size[0] > (1 << 24) || a.q.size[1] > (1 << 20) || a.q.size[2] > (1 << 20) || a.q.size[1] * a.q.size[2] > (1 << 26))
    return SPLASH_ERR_TOO_LARGE;
  return SPLASH_OK;
}

template <typename Shape>
static size_t parts_bytes() {
  return (size_t)resident<Shape>() * 2 * Shape::kRows * (Shape::kV + 2) * 4;
}

static int cache_attend(const SplashCacheAttendArgs& a, cudaStream_t stream) {
  if (const int status = check_attend(a)) return status;
  const SplashKvCache& c = a.cache;
  if (a.workspace == nullptr || (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0) return SPLASH_ERR_INVALID_ARGUMENT;
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
  p.q_heads = (int32_t)a.q.size[1];
  p.kv_heads = c.kv_heads;
  p.heads_per_kv = p.q_heads / c.kv_heads;
  p.q_len = (int32_t)a.q.size[2];
  p.n_table = a.n_table;
  p.page_size = c.page_size;
  p.page_shift = log2_of(c.page_size);
  p.group = c.format == SPLASH_CACHE_INT4 ? c.group : 32;
  p.group_shift = log2_of(p.group);
  p.dtype = a.q.dtype;
  p.head_dim = c.head_dim;
  p.head_dim_v = c.head_dim_v;
  p.window = a.window < 0 ? -1 : a.window;
  return with_shape(a, [&](auto shape) -> int {
    using Shape = decltype(shape);
    const size_t parts = parts_bytes<Shape>();
    if (a.workspace_bytes < parts + 8 * ((size_t)p.batch + 1)) return SPLASH_ERR_INVALID_ARGUMENT;
    AttendParams own = p;
    own.parts = static_cast<float*>(a.workspace);
    own.starts = reinterpret_cast<int64_t*>(static_cast<uint8_t*>(a.workspace) + parts);
    own.row_tiles = (p.q_len * p.heads_per_kv + Shape::kRows - 1) / Shape::kRows;
    own.min_share = kAttendWarps;
    return launch<Shape>(own, resident<Shape>(), stream);
  });
}

static size_t cache_attend_workspace(const SplashCacheAttendArgs& a) {
  if (check_attend(a) != SPLASH_OK) return 0;
  size_t bytes = 0;
  with_shape(a, [&](auto shape) -> int {
    bytes = parts_bytes<decltype(shape)>() + 8 * ((size_t)a.q.size[0] + 1);
    return 0;
  });
  return bytes;
}

}  // namespace sb

extern "C" {

int splash_cache_attend(const SplashCacheAttendArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_attend(*args, static_cast<cudaStream_t>(cuda_stream));
}

size_t splash_cache_attend_workspace_bytes(const SplashCacheAttendArgs* args) {
  return args == nullptr ? 0 : sb::cache_attend_workspace(*args);
}

}  // extern "C"
