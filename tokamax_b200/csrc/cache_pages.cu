// Which pages of the quantised key / value cache a query attends to: bounds of the keys of whole pages, and the choice of those
// whose bounds allow the largest logits.
//
// Mathematics.  With least_c <= k_c <= largest_c for the keys of a page, q . k <= sum over c of max(q_c least_c, q_c largest_c) =
// sum over c of min(q_c, 0) least_c + max(q_c, 0) largest_c, a product of rows of twice the head dim.  Both sides are held in 8 bits, so
// that the sum is one of whole numbers: it has no rounding, and the choice is the same in any order of summation.  (The 8 bits are
// rounded to the nearest: the sum is a score then, a bound within half a step a channel.)  Bounds of a page are 256 bytes a head
// (head dim 128) beside the 9 KB of its keys and values: a choice among all pages costs 3 % of what attention over them would.
#include <atomic>

#include "cache_common.cuh"

namespace sb {

constexpr float kMostCode = 127.f;

// NaN as 0 and infinities as the largest number.
__device__ __forceinline__ float as_number(float x) { return x != x ? 0.f : fminf(fmaxf(x, -3.4028234663852886e38f), 3.4028234663852886e38f); }
// With NaN where an operand is NaN.
__device__ __forceinline__ float least_of(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float largest_of(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Quotients by top / 127, rounded to 32 bits, then to whole numbers in -127 .. 127, as bytes.
struct Coder {
  float scale, inverse;  // (inverse 0: the hardware's own division)
  template <int N>
  __device__ __forceinline__ void operator()(const float (&x)[N], uint32_t (&codes)[(N + 3) / 4]) const {
    constexpr float kUnits = 12582912.f;  // 1.5 * 2^23: a sum is rounded to whole numbers, and has one in its low bits
    float sum[(N + 3) / 4 * 4] = {};
    if (inverse > 0.f) {
#pragma unroll
      for (int j = 0; j < N; ++j) sum[j] = divide(x[j], scale, inverse) + kUnits;
    } else if (scale > 0.f) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float q;
        asm volatile("div.rn.f32 %0, %1, %2;" : "=f"(q) : "f"(x[j]), "f"(scale));  // (volatile: not worked out in any case)
        sum[j] = fminf(fmaxf(q, -kMostCode), kMostCode) + kUnits;
      }
    }
#pragma unroll
    for (int j = 0; j < N; j += 4)
      codes[j / 4] = __byte_perm(__byte_perm(__float_as_uint(sum[j]), __float_as_uint(sum[j + 1]), 0x0040),
                                 __byte_perm(__float_as_uint(sum[j + 2]), __float_as_uint(sum[j + 3]), 0x0040), 0x5410);
  }
};
__device__ __forceinline__ Coder coder_of(float top) {
  const float scale = __fdiv_rn(top, kMostCode);
  const bool exact = scale > kLeastDivisor && (~__float_as_uint(scale) & 0x7fffffu) != 0;
  return {scale, exact ? __frcp_rn(scale) : 0.f};
}

__device__ __forceinline__ bool in_pool(int page, int64_t n_pages) { return page >= 0 && page < n_pages; }

// ------------------------------------------------------------------------------------------
// bounds
// ------------------------------------------------------------------------------------------
struct BoundParams {
  const uint8_t* codes;
  const uint8_t* scales;
  int8_t* bound_codes;
  float* bound_scales;
  const int32_t* page_table;
  const int32_t* lengths;
  int64_t table_stride, n_pages, newest, batch;
  int32_t n_table, page_size, page_shift, kv_heads, head_dim, row, group_shift, split;
};

constexpr int kBoundThreads = 128, kBoundWarps = kBoundThreads / 32;
constexpr int kPiece = 16;  // channels of a lane

// Sixteen channels of a row in 32 bits, from their codes and the scales of their group.
template <int kFormat>
struct RowPiece {
  static constexpr int kBytes = kFormat == SPLASH_CACHE_INT4 ? kPiece / 2 : kPiece;
  uint32_t w[kBytes / 4], scale;
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales) {
    if constexpr (kFormat == SPLASH_CACHE_INT4) {
      const uint2 v = *reinterpret_cast<const uint2*>(codes);
      w[0] = v.x, w[1] = v.y;
      scale = *reinterpret_cast<const uint32_t*>(scales);
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(codes);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      scale = (uint32_t)*reinterpret_cast<const uint16_t*>(scales) << 16;
    }
  }
  __device__ __forceinline__ void get(float (&x)[kPiece]) const {
    const float s = __uint_as_float(scale & 0xffff0000u);
    if constexpr (kFormat == SPLASH_CACHE_INT4) {
      // A code that stands 4 i bits up in a word is that of 2^(23 - 4 i) + code, for i up to 4: a mask and an exponent, one instruction.
      // (Zero and product are 8 and 12 bits, their sum is rounded once.)
      const float zero = bf16_bits_to_float(scale);
#pragma unroll
      for (int j = 0; j < kPiece; ++j) {
        const int i = j % 8 < 5 ? j % 8 : j % 8 - 5;
        const uint32_t word = j % 8 < 5 ? w[j / 8] : w[j / 8] >> 20, exponent = 0x4b000000u - i * 0x02000000u;
        uint32_t above;  // (the compiler takes two instructions for it)
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(above) : "r"(word), "r"(15u << 4 * i), "r"(exponent));
        x[j] = fmaf(s, __uint_as_float(above) - __uint_as_float(exponent), zero);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPiece / 2; ++j) {
        const uint32_t pair = e4m3x2_to_f16x2(w[j / 2] >> (16 * (j & 1)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        x[2 * j] = s * f.x;
        x[2 * j + 1] = s * f.y;
      }
    }
  }
};

constexpr int kWarpTokens = 64;

// Bound by instructions and latency, not by memory (72 bytes a row of 128 channels in four bits): a channel of a key takes an extraction
// (a mask with an exponent, 2 cycles of a scheduler), a sum, a fused multiply-add and two extremes, 6.1 cycles, and a page some 500
// instructions beside.  A warp a page of 64 tokens, eight rows a lane in flight: 4 prompts of up to 8192 tokens, 8 heads of 128, 8.0 us (26
// with a block of 256 threads a page and its extremes by way of shared memory, 9.6 with quotients of 64 bits for pages and heads and two
// instructions for an extraction, 8.6 with four rows in flight, 10.3 with 32 tokens a warp); the instructions alone 3.6, memory 1.6.
// Eight channels a lane, 16 to 32 warps on an SM, sums of two channels in an instruction: no faster.  e4m3 rows are twice as wide: eight in flight
// spill 88 to 100 bytes a thread (3 x 517 tokens behind 1999 .. 6001, 3.5 us).
// `split` warps of a block have a page of a sequence and kv head; blockIdx.x: the page (from the first that has become whole), y: the
// sequence, z: kv heads.  A team of kTeam lanes (the power of two that holds the row's width / 16) has a
// token's row.
template <int kFormat, int kTeam>
__global__ void __launch_bounds__(kBoundThreads, 4) cache_bound_kernel(const __grid_constant__ BoundParams p) {
  constexpr int kRows = 32 / kTeam;       // of a warp's load
  constexpr int kAhead = 8;               // loads in flight
  constexpr int kOwn = kPiece / kRows;    // channels of a lane once the rows are together
  static_assert(kOwn >= 2);
  __shared__ float extremes[kBoundWarps][2][32 * kOwn];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane % kTeam, team = lane / kTeam;
  const int share = warp & (p.split - 1);  // of the page's tokens (`split` is a power of two)
  const int head = (int)((blockIdx.z * blockDim.x + threadIdx.x) / (32u * p.split));
  const bool real = part * kPiece < p.row;  // (of teams of 96 and 192 channels some lanes have none)
  for (int64_t b = blockIdx.y; b < p.batch; b += gridDim.y) {
    const int64_t length = min((int64_t)max(__ldg(p.lengths + b), 0), (int64_t)p.n_table << p.page_shift);
    const int64_t first = max(length - p.newest, (int64_t)0) >> p.page_shift, whole = length >> p.page_shift;
    const int64_t index = first + blockIdx.x;
    if (index < whole) {  // (all warps of the block alike)
      const int page = head < p.kv_heads ? __ldg(p.page_table + b * p.table_stride + index) : -1;
      const bool mine = in_pool(page, p.n_pages);
      float lo[kPiece], hi[kPiece];
#pragma unroll
      for (int j = 0; j < kPiece; ++j) lo[j] = INFINITY, hi[j] = -INFINITY;
      const uint32_t row0 = ((uint32_t)max(page, 0) * p.kv_heads + head) << p.page_shift;
      const int row_bytes = kFormat == SPLASH_CACHE_INT4 ? p.row / 2 : p.row, scale_bytes = kFormat == SPLASH_CACHE_INT4 ? (p.row >> p.group_shift) * 4 : 2;
      const uint8_t* const codes = p.codes + (uint64_t)row0 * (unsigned)row_bytes + part * RowPiece<kFormat>::kBytes;
      const uint8_t* const scales = p.scales + (uint64_t)row0 * (unsigned)scale_bytes + (kFormat == SPLASH_CACHE_INT4 ? (part * kPiece >> p.group_shift) * 4 : 0);
      const int own_tokens = p.page_size / p.split, t0 = share * own_tokens + team, t1 = (share + 1) * own_tokens;
      auto each = [&](auto&& take) {  // of the lane's tokens, kAhead at a time
        for (int t = t0; t < t1; t += kRows * kAhead) {
          RowPiece<kFormat> piece[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i)  // (tokens come in sixteens: two of a lane's at least)
            if (t + i * kRows < t1) piece[i].load(codes + (int64_t)(t + i * kRows) * row_bytes, scales + (int64_t)(t + i * kRows) * scale_bytes);
#pragma unroll
          for (int i = 0; i < kAhead; i += 2) {
            if (t + i * kRows >= t1) break;
            float x[kPiece], y[kPiece];
            piece[i].get(x);
            piece[i + 1].get(y);
#pragma unroll
            for (int j = 0; j < kPiece; ++j) take(j, x[j], y[j]);
          }
        }
      };
      if (mine && real) {
        each([&](int j, float x, float y) {
          lo[j] = least_of(lo[j], x, y);
          hi[j] = largest_of(hi[j], x, y);
        });
        // What is no number or an infinity shows in the extremes: a second look takes it for what it counts as.
        bool plain = true;
#pragma unroll
        for (int j = 0; j < kPiece; ++j) plain = plain && lo[j] > -INFINITY && hi[j] < INFINITY;  // (not where one is NaN)
        if (!plain) {
#pragma unroll
          for (int j = 0; j < kPiece; ++j) lo[j] = INFINITY, hi[j] = -INFINITY;
          each([&](int j, float x, float y) {
            lo[j] = least_of(lo[j], as_number(x), as_number(y));
            hi[j] = largest_of(hi[j], as_number(x), as_number(y));
          });
        }
      }
      // The rows of a warp's load together: at each step a lane keeps half of its channels.
#pragma unroll
      for (int d = kTeam, n = kPiece / 2; d < 32; d <<= 1, n >>= 1) {
        const bool upper = lane & d;
#pragma unroll
        for (int j = 0; j < n; ++j) {
          const float give_lo = upper ? lo[j] : lo[j + n], give_hi = upper ? hi[j] : hi[j + n];
          lo[j] = fminf(upper ? lo[j + n] : lo[j], __shfl_xor_sync(~0u, give_lo, d));
          hi[j] = fmaxf(upper ? hi[j + n] : hi[j], __shfl_xor_sync(~0u, give_hi, d));
        }
      }
      if (p.split > 1) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) extremes[warp][0][j * 32 + lane] = lo[j], extremes[warp][1][j * 32 + lane] = hi[j];
        __syncthreads();
        if (share == 0) {
          for (int w = warp + 1; w < warp + p.split; ++w)
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
              lo[j] = fminf(lo[j], extremes[w][0][j * 32 + lane]);
              hi[j] = fmaxf(hi[j], extremes[w][1][j * 32 + lane]);
            }
        }
        __syncthreads();
      }
      if (share != 0 || !mine) continue;  // (whole warps)
      // the lane's channels: kOwn from part * 16 on, and those that it gave away before them
      int channel = part * kPiece;
#pragma unroll
      for (int d = kTeam, n = kPiece / 2; d < 32; d <<= 1, n >>= 1) channel += lane & d ? n : 0;
      float top = 0.f, lo_own[kOwn], hi_own[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        lo_own[j] = channel + j < p.head_dim ? lo[j] : 0.f;
        hi_own[j] = channel + j < p.head_dim ? hi[j] : 0.f;
        top = fmaxf(top, fmaxf(fabsf(lo_own[j]), fabsf(hi_own[j])));
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      const Coder code = coder_of(top);
      const uint64_t at = (uint64_t)((uint32_t)page * p.kv_heads + head);
      if (real) {
        int8_t* const to = p.bound_codes + at * (unsigned)(2 * p.row) + channel;
        uint32_t least[(kOwn + 3) / 4], largest[(kOwn + 3) / 4];
        code(lo_own, least);
        code(hi_own, largest);
        if constexpr (kOwn == 2) {
          *reinterpret_cast<uint16_t*>(to) = (uint16_t)least[0];
          *reinterpret_cast<uint16_t*>(to + p.row) = (uint16_t)largest[0];
        } else {
#pragma unroll
          for (int j = 0; j < kOwn / 4; ++j) {
            *reinterpret_cast<uint32_t*>(to + 4 * j) = least[j];
            *reinterpret_cast<uint32_t*>(to + p.row + 4 * j) = largest[j];
          }
        }
      }
      if (lane == 0) p.bound_scales[at] = code.scale;
    }
  }
}

static int check_bounds(const SplashPageBounds& b) {
  return b.codes == nullptr || (reinterpret_cast<uintptr_t>(b.codes) & 15u) != 0 || b.scales == nullptr ||
                 (reinterpret_cast<uintptr_t>(b.scales) & 3u) != 0
             ? SPLASH_ERR_INVALID_ARGUMENT
             : SPLASH_OK;
}

static int check_pages(const SplashKvCache& c, const int32_t* table, const int32_t* lengths, int32_t n_table, int64_t stride) {
  if (table == nullptr || lengths == nullptr || n_table <= 0 || stride < 0) return SPLASH_ERR_INVALID_ARGUMENT;
  return (int64_t)n_table * c.page_size > (1 << 30) ? SPLASH_ERR_TOO_LARGE : SPLASH_OK;
}

static int cache_bound(const SplashCacheBoundArgs& a, cudaStream_t stream) {
  const SplashKvCache& c = a.cache;
  if (const int status = check_cache(c)) return status;
  if (const int status = check_bounds(a.bounds)) return status;
  if (const int status = check_pages(c, a.page_table, a.lengths, a.n_table, a.table_stride)) return status;
  if (a.batch <= 0 || a.newest < 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.batch > (1 << 24)) return SPLASH_ERR_TOO_LARGE;
  if (a.newest == 0) return SPLASH_OK;
  BoundParams p{};
  p.codes = static_cast<const uint8_t*>(c.k_codes);
  p.scales = static_cast<const uint8_t*>(c.k_scales);
  p.bound_codes = a.bounds.codes;
  p.bound_scales = a.bounds.scales;
  p.page_table = a.page_table;
  p.lengths = a.lengths;
  p.table_stride = a.table_stride;
  p.n_pages = c.n_pages;
  p.newest = a.newest;
  p.batch = a.batch;
  p.n_table = a.n_table;
  p.page_size = c.page_size;
  p.page_shift = log2_of(c.page_size);
  p.kv_heads = c.kv_heads;
  p.head_dim = c.head_dim;
  p.row = c.row_k;
  p.group_shift = log2_of(c.group);
  // n tokens make n / page_size + 1 pages whole at most
  const int64_t pages = a.newest / c.page_size + 1;
  // A warp has up to kWarpTokens of a page's tokens, as far as the warps of a block go.
  p.split = 1;
  while (p.split < kBoundWarps && p.split * kWarpTokens < c.page_size) p.split *= 2;
  const int most = kBoundWarps / p.split, heads = c.kv_heads < most ? c.kv_heads : most;  // of a block
  const dim3 grid((unsigned)(pages < a.n_table ? pages : a.n_table), (unsigned)(a.batch < 65535 ? a.batch : 65535),
                  (unsigned)((c.kv_heads + heads - 1) / heads));
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attribute = early_launch();
  config.gridDim = grid;
  config.blockDim = dim3(heads * p.split * 32);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  auto launch = [&](auto format) {
    constexpr int kFormat = decltype(format)::value;
    return c.row_k <= 64    ? cudaLaunchKernelEx(&config, cache_bound_kernel<kFormat, 4>, p)
           : c.row_k <= 128 ? cudaLaunchKernelEx(&config, cache_bound_kernel<kFormat, 8>, p)
                            : cudaLaunchKernelEx(&config, cache_bound_kernel<kFormat, 16>, p);
  };
  const cudaError_t launched = c.format == SPLASH_CACHE_INT4 ? launch(std::integral_constant<int, SPLASH_CACHE_INT4>{})
                                                             : launch(std::integral_constant<int, SPLASH_CACHE_E4M3>{});
  return launched == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

// A thread has eight channels of one side of a page and head.
__global__ void __launch_bounds__(kBoundThreads) cache_bound_values_kernel(const int8_t* codes, const float* scales, float* out, uint32_t sides,
                                                                           int row, int vectors) {
  const uint64_t step = (uint64_t)gridDim.x * kBoundThreads, all = (uint64_t)sides * (unsigned)vectors;
  for (uint64_t at = (uint64_t)blockIdx.x * kBoundThreads + threadIdx.x; at < all; at += step) {
    const uint32_t side = (uint32_t)(all >> 32 == 0 ? (uint32_t)at / (unsigned)vectors : at / (unsigned)vectors);
    const uint32_t part = (uint32_t)(at - (uint64_t)side * (unsigned)vectors);
    const float scale = __ldg(scales + side / 2);
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(codes + (uint64_t)side * (unsigned)row + part * 8));
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = scale * (float)(int8_t)((j < 4 ? w.x : w.y) >> 8 * (j % 4) & 255u);
    store8(out, SPLASH_F32, (int64_t)(at * 8), x);
  }
}

static int cache_bound_values(const SplashKvCache& c, const SplashPageBounds& bounds, float* values, cudaStream_t stream) {
  if (const int status = check_cache(c)) return status;
  if (const int status = check_bounds(bounds)) return status;
  if (values == nullptr || (reinterpret_cast<uintptr_t>(values) & 15u) != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  const int64_t sides = c.n_pages * c.kv_heads * 2, blocks = (sides * (c.head_dim / 8) + kBoundThreads - 1) / kBoundThreads;
  cache_bound_values_kernel<<<(unsigned)(blocks < kSms * 16 ? blocks : kSms * 16), kBoundThreads, 0, stream>>>(bounds.codes, bounds.scales, values,
                                                                                                         (uint32_t)sides, c.row_k, c.head_dim / 8);
  return cudaGetLastError() == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

// ------------------------------------------------------------------------------------------
// the choice
// ------------------------------------------------------------------------------------------
struct ChooseParams {
  const int8_t* bound_codes;
  const float* bound_scales;
  const void* q;
  const int32_t* page_table;
  const int32_t* lengths;
  int32_t* tables;
  int32_t* table_lengths;
  uint32_t* keys;  // scores of a row's pages, [rows][n_table], where shared memory has no room for them; else NULL
  int64_t q_stride_b, q_stride_h, q_stride_s, table_stride, n_pages;
  int32_t dtype, kv_heads, heads_per_kv, q_len, n_table, page_size, page_shift, head_dim, row, count, first, last;
};

constexpr int kKeysOnChip = 8192;         // pages of a row whose scores, and numbers, shared memory holds
constexpr int kMostHeads = 128;           // q heads of a kv head
constexpr int kMostCluster = 8, kMostChooseWarps = 8, kFewPages = 1024;
constexpr int kBins = 1024, kBinBits = 10;
constexpr int kFew = 64;  // keys that are counted against each other
// Scores as unsigned numbers of the same order; 0: no candidate, kAlways: taken before all others.
constexpr uint32_t kNoCandidate = 0, kAlways = ~0u;
__device__ __forceinline__ uint32_t key_of(float score) {
  const uint32_t bits = score == score ? __float_as_uint(score + 0.f) : 0u;  // (-0 and NaN, of bounds that nobody wrote, as 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Products of rows of 8-bit numbers, 16 x 32 by 32 x 8, added to c.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory of a CTA: q's codes [heads, to a multiple of 8][2 * row, and 64 bytes], then the keys and the pages' numbers
// (of the cluster's first CTA).
__host__ __device__ constexpr int choose_pitch(int row) { return 2 * row + 64; }
__host__ __device__ constexpr int choose_heads(int heads) { return (heads + 7) / 8 * 8; }

struct Found {  // of a row's pages
  uint32_t least, most;  // keys but for kAlways
  int candidates, always;
};

// A cluster (of one CTA and more) has a query and kv head: its CTAs score pages, tile by tile of 16, and the first one chooses.
// The bounds of a page are a row of the products' first operand as they lie in memory: channels may come in any order as long as q's do
// too, so that a lane's 16 bytes are the registers of two products.  The wanted-th largest of the scores is found by a histogram of
// 1024 bins over their range; the few in its bin are counted against each other.
// Bound by latency: of some 13000 cycles for 2048 pages, 8 CTAs a row (7.4 us) the first loads take 2000, q's codes 1600, two tiles of each
// warp 2400, the cluster's barrier 1300, the histogram 1600, the few 2200 and the writing 1700, all of it chains of dependent steps at 20 % of
// the instructions that an SM could issue.  32 sequences of 8192 .. 32768 tokens 9.5 us (21 MB of bounds: 3.3).  Tried: tiles through
// shared memory by asynchronous copies 11.5, two and three tiles ahead 10.5, 8 warps for short rows (62 pages, 512 rows) 6.2 -> 10.2.
// kChunks: pieces of 64 numbers that the bounds of a page are; kOnChip: the scores are in shared memory.
template <int kChunks, int kWarps, bool kOnChip>
__global__ void __launch_bounds__(kWarps * 32, (kChunks <= 4 ? 16 : 8) / kWarps) cache_choose_kernel(const __grid_constant__ ChooseParams p) {
  constexpr int kThreads = kWarps * 32, kRow = kChunks * 32, kPitch = choose_pitch(kRow);
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) Found found;
  __shared__ __align__(16) uint32_t bins[kBins];
  __shared__ __align__(16) uint2 few[kFew];  // keys and their places
  __shared__ __align__(16) uint32_t tops[kWarps], sums[kWarps];
  __shared__ uint32_t counts[kWarps][2], picked[3], few_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  uint32_t ctas, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const uint32_t row = blockIdx.x / ctas;  // (sequence, kv head, query)
  const int i = row % (unsigned)p.q_len, head = row / (unsigned)p.q_len % (unsigned)p.kv_heads, b = row / (unsigned)p.q_len / (unsigned)p.kv_heads;
  grid_dependency_wait();
  const int length = __ldg(p.lengths + b);

  // ---- a warp's tiles: 16 pages each, their bounds as operands of the products ----
  const int32_t* const table = p.page_table + b * p.table_stride;
  const int step = (int)ctas * kWarps * 16;
  const int first = ((int)rank + warp * (int)ctas) * 16;
  // Numbers of pages for two tiles at a time: lane i has page i % 16 of tile turn + i / 16 (behind the table: not looked at).
  auto look_up = [&](int turn) { return __ldg(table + min(first + (turn + (lane >> 4)) * step + (lane & 15), p.n_table - 1)); };
  int numbers_now = look_up(0), numbers_next = look_up(2);
  struct Tile {
    uint4 a[kChunks], a8[kChunks];  // of rows g and g + 8
    float scale;                    // of lanes 0 and 1 of four: row g's and row g + 8's
    int page;                       // the same
  };
  auto load_tile = [&](Tile& tile, int numbers, int which) {  // (what is no candidate is read as page 0)
    const int page0 = __shfl_sync(~0u, numbers, which * 16 + g), page1 = __shfl_sync(~0u, numbers, which * 16 + 8 + g);
    const uint32_t at0 = (uint32_t)(in_pool(page0, p.n_pages) ? page0 : 0) * p.kv_heads + head;
    const uint32_t at1 = (uint32_t)(in_pool(page1, p.n_pages) ? page1 : 0) * p.kv_heads + head;
    const uint4* const from0 = reinterpret_cast<const uint4*>(p.bound_codes + (uint64_t)at0 * (2 * kRow)) + t4;
    const uint4* const from1 = reinterpret_cast<const uint4*>(p.bound_codes + (uint64_t)at1 * (2 * kRow)) + t4;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) tile.a[k] = __ldg(from0 + k * 4), tile.a8[k] = __ldg(from1 + k * 4);
    tile.scale = __ldg(p.bound_scales + (t4 & 1 ? at1 : at0));
    tile.page = t4 & 1 ? page1 : page0;
  };
  // a thread has eight channels of every kThreads / (kRow / 8)-th head; the first head's stay with it
  constexpr int kVectors = kRow / 8, kAtOnce = kThreads / kVectors;
  const int vectors = p.head_dim / 8, heads = choose_heads(p.heads_per_kv), d = tid % kVectors, h_first = tid / kVectors;
  const bool in_row = d < vectors && h_first < kAtOnce;
  const uint16_t* const q = static_cast<const uint16_t*>(p.q) + b * p.q_stride_b + (int64_t)head * p.heads_per_kv * p.q_stride_h + i * p.q_stride_s;
  auto load_q = [&](int h) {  // (rows that make up eight repeat the first one)
    return __ldg(reinterpret_cast<const uint4*>(q + (h < p.heads_per_kv ? h : 0) * p.q_stride_h + d * 8));
  };
  uint4 q_first = make_uint4(0, 0, 0, 0);
  if (in_row) q_first = load_q(h_first);
  for (int k = tid * 4; k < kBins; k += kThreads * 4) *reinterpret_cast<uint4*>(bins + k) = make_uint4(0, 0, 0, 0);
  if (tid == 0) {
    few_count = 0;
    found = {~0u, 0u, 0, 0};
  }
  __syncwarp();
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const int64_t reach = (int64_t)p.n_table << p.page_shift;
  const int position = (int)min(max((int64_t)length - p.q_len + i, (int64_t)-1), reach - 1);
  const int own = position >> p.page_shift, pages = own + 1;  // (-1 and 0 before the sequence)

  // ---- q in 8 bits ----
  auto numbers = [&](const uint4& w, float (&x)[8]) {
    unpack16(p.dtype, w.x, x[0], x[1]);
    unpack16(p.dtype, w.y, x[2], x[3]);
    unpack16(p.dtype, w.z, x[4], x[5]);
    unpack16(p.dtype, w.w, x[6], x[7]);
  };
  auto top_of = [&](const uint4& w) {  // the largest size as bits, which sizes are in the order of; infinity for what is no number
    float x[8], top = 0.f;
    numbers(w, x);
#pragma unroll
    for (int k = 0; k < 8; k += 2) top = largest_of(top, fabsf(x[k]), fabsf(x[k + 1]));
    return min(__float_as_uint(top), 0x7f800000u);
  };
  uint32_t top = top_of(q_first);
  if (in_row)
    for (int h = h_first + kAtOnce; h < p.heads_per_kv; h += kAtOnce) top = max(top, top_of(load_q(h)));
  top = __reduce_max_sync(~0u, top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = max(top, tops[w]);
  const bool finite = top < 0x7f800000u;
  if (!finite) {  // (all threads alike) once more, with each number as what it counts as
    float most = 0.f;
    if (in_row)
      for (int h = h_first; h < p.heads_per_kv; h += kAtOnce) {
        float x[8];
        numbers(load_q(h), x);
#pragma unroll
        for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(as_number(x[k])));
      }
    __syncthreads();
    top = __reduce_max_sync(~0u, __float_as_uint(most));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max(top, tops[w]);
  }
  Tile tile;
  if (first < pages) load_tile(tile, numbers_now, 0);
  const Coder coder = coder_of(__uint_as_float(top));
  if (h_first < kAtOnce) {
    for (int h = h_first; h < heads; h += kAtOnce) {
      uint32_t negative[2] = {0, 0}, positive[2] = {0, 0};
      if (d < vectors) {
        float x[8];
        uint32_t codes[2];
        numbers(h == h_first ? q_first : load_q(h), x);
        if (!finite) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = as_number(x[k]);
        }
        coder(x, codes);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t below;  // of each byte its sign
          asm("prmt.b32 %0, %1, 0, 0xba98;" : "=r"(below) : "r"(codes[k]));
          negative[k] = codes[k] & below;
          positive[k] = codes[k] & ~below;
        }
      }
      *reinterpret_cast<uint2*>(smem + h * kPitch + d * 8) = make_uint2(negative[0], negative[1]);
      *reinterpret_cast<uint2*>(smem + h * kPitch + kRow + d * 8) = make_uint2(positive[0], positive[1]);
    }
  }
  __syncthreads();

  // ---- scores ----
  uint32_t* own_keys;  // and, in shared memory, the pages' numbers behind them
  if constexpr (kOnChip)
    own_keys = reinterpret_cast<uint32_t*>(smem + heads * kPitch);
  else
    own_keys = p.keys + (uint64_t)row * p.n_table;
  uint32_t* to_keys = own_keys;
  Found* to_found = &found;
  if (ctas > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // (the first CTA is there)
    uint64_t at;
    if constexpr (kOnChip) {
      asm("mapa.u64 %0, %1, 0;" : "=l"(at) : "l"(reinterpret_cast<uint64_t>(own_keys)));
      to_keys = reinterpret_cast<uint32_t*>(at);
    }
    asm("mapa.u64 %0, %1, 0;" : "=l"(at) : "l"(reinterpret_cast<uint64_t>(to_found)));
    to_found = reinterpret_cast<Found*>(at);
  }
  uint32_t least = ~0u, most = 0;
  int candidates = 0, always = 0;
  for (int turn = 0, at = first; at < pages; ++turn, at += step) {
    Tile next;
    if (at + step < pages) load_tile(next, turn & 1 ? numbers_next : numbers_now, ~turn & 1);
    if (turn & 1) {
      numbers_now = numbers_next;
      numbers_next = look_up(turn + 3);
    }
    int best0 = INT32_MIN, best1 = INT32_MIN;
    for (int h0 = 0; h0 < heads; h0 += 8) {
      const uint8_t* const codes = smem + (h0 + g) * kPitch + t4 * 16;
      int c[2][4] = {};  // (two chains)
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const uint4 w = *reinterpret_cast<const uint4*>(codes + k * 64), &a = tile.a[k], &a8 = tile.a8[k];
        mma_s8(c[0], a.x, a8.x, a.y, a8.y, w.x, w.y);
        mma_s8(c[1], a.z, a8.z, a.w, a8.w, w.z, w.w);
      }
      best0 = max(best0, max(c[0][0] + c[1][0], c[0][1] + c[1][1]));
      best1 = max(best1, max(c[0][2] + c[1][2], c[0][3] + c[1][3]));
    }
    // lanes 0 and 1 of four have a page each
    best0 = max(best0, __shfl_xor_sync(~0u, best0, 2));
    best1 = max(best1, __shfl_xor_sync(~0u, best1, 2));
    int best = t4 & 1 ? best1 : best0;
    best = max(best, __shfl_xor_sync(~0u, t4 & 1 ? best0 : best1, 1));
    const int index = at + (t4 & 1) * 8 + g;
    if (t4 < 2 && index < pages) {
      uint32_t key = key_of((float)best * tile.scale);
      if (!in_pool(tile.page, p.n_pages)) {
        key = kNoCandidate;
      } else if (index < p.first || index > own - p.last) {
        key = kAlways;
        ++always;
        ++candidates;
      } else {
        least = min(least, key);
        most = max(most, key);
        ++candidates;
      }
      to_keys[index] = key;
      if constexpr (kOnChip) to_keys[p.n_table + index] = (uint32_t)tile.page;
    }
    tile = next;
  }
  __syncwarp();
  least = __reduce_min_sync(~0u, least);
  most = __reduce_max_sync(~0u, most);
  candidates = __reduce_add_sync(~0u, candidates);
  always = __reduce_add_sync(~0u, always);
  if (lane == 0 && candidates > 0) {
    atomicMin(&to_found->least, least);
    atomicMax(&to_found->most, most);
    atomicAdd(&to_found->candidates, candidates);
    atomicAdd(&to_found->always, always);
  }
  __syncwarp();
  if (ctas > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // ---- which are taken: keys whose difference from the least, without its low bits, is above `prefix`, and of those that are equal
  // to it the first `equal` ones ----
  const Found all_found = found;
  uint32_t prefix = 0;
  int bits = 32, equal = INT32_MAX;  // (all)
  // of eight keys, kThreads (or 32) apart
  auto load_keys = [&](int at, int until, int apart, uint32_t (&keys)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) keys[k] = at + k * apart < until ? own_keys[at + k * apart] : kNoCandidate;
  };
  auto ranked = [](uint32_t key) { return key != kNoCandidate && key != kAlways; };
  auto high_of = [&](uint32_t key) { return bits == 32 ? 0u : (key - all_found.least) >> bits; };
  bool by_few = false;
  if (all_found.candidates > p.count) {
    int wanted = p.count - all_found.always;  // of the ranked ones; fewer than there are
    equal = 0;
    prefix = ~0u;  // (none of them)
    bits = 0;
    if (wanted > 0) {
      // Digits of the difference, from the highest: of each the bin that the wanted-th largest key lies in.
      bits = 32 - __clz(all_found.most - all_found.least);
      prefix = 0;
      while (true) {
        const int shift = max(bits - kBinBits, 0);
        const uint32_t mask = (1u << (bits - shift)) - 1;
        for (int at = tid; at < pages; at += kThreads * 8) {
          uint32_t keys[8];
          load_keys(at, pages, kThreads, keys);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (ranked(keys[k]) && high_of(keys[k]) == prefix) atomicAdd(&bins[(keys[k] - all_found.least) >> shift & mask], 1u);
        }
        __syncthreads();
        // bins from the highest, kEach a thread
        constexpr int kEach = kBins / kThreads;
        uint32_t each[kEach], sum = 0;
#pragma unroll
        for (int k = 0; k < kEach; k += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(bins + kBins - 4 - k - kEach * tid);
          each[k] = v.w, each[k + 1] = v.z, each[k + 2] = v.y, each[k + 3] = v.x;
          sum += v.x + v.y + v.z + v.w;
        }
        uint32_t before = sum;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const uint32_t other = __shfl_up_sync(~0u, before, s);
          if (lane >= s) before += other;
        }
        if (lane == 31) sums[warp] = before;
        __syncthreads();
        before -= sum;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) before += w < warp ? sums[w] : 0;
        if (before < (uint32_t)wanted && before + sum >= (uint32_t)wanted) {
#pragma unroll
          for (int k = 0; k < kEach; ++k) {
            if (before < (uint32_t)wanted && before + each[k] >= (uint32_t)wanted) {
              picked[0] = kBins - 1 - kEach * tid - k;
              picked[1] = before;
              picked[2] = each[k];
            }
            before += each[k];
          }
        }
        __syncthreads();
        prefix = prefix << (bits - shift) | picked[0];
        wanted -= (int)picked[1];
        bits = shift;
        const int population = (int)picked[2];
        by_few = population > wanted && population <= kFew;
        if (bits == 0 || population <= kFew || population == wanted) break;
        for (int k = tid; k < kBins; k += kThreads) bins[k] = 0;
        __syncthreads();
      }
      equal = wanted;
    }
  }

  // ---- how many, and where: a warp has a run of pages ----
  const int run = (pages + kThreads - 1) / kThreads * 32, from = min(warp * run, pages), until = min(from + run, pages);
  const uint32_t below = (1u << lane) - 1;
  uint32_t taken[8], alike[8];
  auto look = [&](int at, uint32_t (&keys)[8]) {
    load_keys(at + lane, until, 32, keys);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t high = high_of(keys[k]);
      taken[k] = __ballot_sync(~0u, keys[k] == kAlways || (ranked(keys[k]) && high > prefix));
      alike[k] = __ballot_sync(~0u, ranked(keys[k]) && high == prefix);
    }
  };
  uint32_t n_taken = 0, n_alike = 0, keys[8];
  for (int at = from; at < until; at += 256) {
    look(at, keys);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      n_taken += __popc(taken[k]);
      n_alike += __popc(alike[k]);
      if (by_few && alike[k] >> lane & 1) few[atomicAdd(&few_count, 1u)] = make_uint2(keys[k], at + k * 32 + lane);
    }
  }
  if (lane == 0) counts[warp][0] = n_taken, counts[warp][1] = by_few ? 0 : n_alike;
  __syncthreads();
  if (by_few) {  // a few that differ in lower bits are counted against each other; those taken are marked
    const int population = (int)few_count;
    if (tid < population) {
      const uint2 mine = few[tid];
      int above = 0;
      for (int k = 0; k < population; ++k) {
        const uint2 other = few[k];
        above += other.x > mine.x || (other.x == mine.x && other.y < mine.y);
      }
      if (above < equal) {
        own_keys[mine.y] = kAlways;
        atomicAdd(&counts[mine.y / run][0], 1u);
      }
    }
    equal = 0;
    __syncthreads();
  }
  int place = 0, alikes = 0, all = 0, all_alike = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    place += w < warp ? (int)counts[w][0] : 0;
    alikes += w < warp ? (int)counts[w][1] : 0;
    all += (int)counts[w][0];
    all_alike += (int)counts[w][1];
  }
  all += min(all_alike, equal);
  int32_t* const to = p.tables + (uint64_t)row * p.count;
  for (int at = from; at < until; at += 256) {
    if (run > 256) look(at, keys);  // (else they are there)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int index = at + k * 32 + lane;
      if (by_few && alike[k] != 0) taken[k] |= __ballot_sync(~0u, alike[k] >> lane & 1 && own_keys[index] == kAlways);
      const int alike_before = alikes + __popc(alike[k] & below);
      if (taken[k] >> lane & 1 || (alike[k] >> lane & 1 && alike_before < equal))
        to[place + __popc(taken[k] & below) + min(alike_before, equal)] = kOnChip ? (int)own_keys[p.n_table + index] : __ldg(table + index);
      place += __popc(taken[k]);
      alikes += __popc(alike[k]);
    }
  }
  for (int k = all + tid; k < p.count; k += kThreads) to[k] = -1;
  if (tid == 0) {
    // the query's own page, the last one, is there up to the query
    const bool has_own = pages > 0 && own_keys[own] != kNoCandidate;
    p.table_lengths[row] = (all << p.page_shift) - (has_own ? p.page_size - 1 - (position & (p.page_size - 1)) : 0);
  }
}

static int check_choose(const SplashCacheChooseArgs& a) {
  const SplashKvCache& c = a.cache;
  if (const int status = check_cache(c)) return status;
  if (const int status = check_bounds(a.bounds)) return status;
  if (const int status = check_cache_tensor(a.q, false)) return status;
  if (const int status = check_pages(c, a.page_table, a.lengths, a.n_table, a.table_stride)) return status;
  if (a.q.size[3] != c.head_dim || a.q.size[1] % c.kv_heads != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.tables == nullptr || a.table_lengths == nullptr) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.first < 0 || a.last < 1 || (int64_t)a.first + a.last > a.count) return SPLASH_ERR_INVALID_ARGUMENT;
  // (as splash_cache_attend_tables takes them; rows of q that shared memory has room for)
  if (a.q.size[0] > (1 << 24) || a.q.size[2] > (1 << 20) || a.q.size[0] * c.kv_heads * a.q.size[2] > (1 << 24) ||
      (int64_t)a.count * c.page_size > (1 << 30) || a.q.size[1] / c.kv_heads > kMostHeads)
    return SPLASH_ERR_TOO_LARGE;
  return SPLASH_OK;
}

static size_t choose_workspace(const SplashCacheChooseArgs& a) {
  if (check_choose(a) != SPLASH_OK) return 0;
  if (a.n_table <= kKeysOnChip) return 0;
  return (size_t)(a.q.size[0] * a.cache.kv_heads * a.q.size[2]) * a.n_table * sizeof(uint32_t);
}

template <int kChunks, int kWarps, bool kOnChip>
static int launch_choose(const cudaLaunchConfig_t& config, const ChooseParams& p) {
  const auto kernel = cache_choose_kernel<kChunks, kWarps, kOnChip>;
  constexpr int kMostShared = kMostHeads * choose_pitch(kChunks * 32) + (kOnChip ? kKeysOnChip * 8 : 0);
  static_assert(kMostShared + 8 * 1024 <= 227 * 1024);
  static std::atomic<uint64_t> ready{0};  // devices that know how much shared memory the kernel takes
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return SPLASH_ERR_CUDA;
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return SPLASH_ERR_CUDA;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  return cudaLaunchKernelEx(&config, kernel, p) == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

static int cache_choose(const SplashCacheChooseArgs& a, cudaStream_t stream) {
  if (const int status = check_choose(a)) return status;
  const SplashKvCache& c = a.cache;
  ChooseParams p{};
  if (const size_t bytes = choose_workspace(a)) {
    if (a.workspace == nullptr || (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0 || a.workspace_bytes < bytes) return SPLASH_ERR_INVALID_ARGUMENT;
    p.keys = static_cast<uint32_t*>(a.workspace);
  }
  p.bound_codes = a.bounds.codes;
  p.bound_scales = a.bounds.scales;
  p.q = a.q.data;
  p.page_table = a.page_table;
  p.lengths = a.lengths;
  p.tables = a.tables;
  p.table_lengths = a.table_lengths;
  p.q_stride_b = a.q.stride[0], p.q_stride_h = a.q.stride[1], p.q_stride_s = a.q.stride[2];
  p.table_stride = a.table_stride;
  p.n_pages = c.n_pages;
  p.dtype = a.q.dtype;
  p.kv_heads = c.kv_heads;
  p.heads_per_kv = (int32_t)(a.q.size[1] / c.kv_heads);
  p.q_len = (int32_t)a.q.size[2];
  p.n_table = a.n_table;
  p.page_size = c.page_size;
  p.page_shift = log2_of(c.page_size);
  p.head_dim = c.head_dim;
  p.row = c.row_k;
  p.count = a.count;
  p.first = a.first;
  p.last = a.last;
  const int64_t rows = a.q.size[0] * c.kv_heads * a.q.size[2];
  // As many CTAs a row as the GPU has room for, each with a tile for each of its warps.
  const int warps = a.n_table <= kFewPages ? kMostChooseWarps / 2 : kMostChooseWarps;
  int ctas = 1;
  while (ctas < kMostCluster && rows * ctas * 2 <= 2 * kSms && (int64_t)a.n_table > (int64_t)ctas * warps * 16) ctas *= 2;
  const int smem = choose_heads(p.heads_per_kv) * choose_pitch(p.row) + (p.keys == nullptr ? a.n_table * 8 : 0);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(rows * ctas));
  config.blockDim = dim3(warps * 32);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2]{early_launch(), cluster_size(ctas)};
  config.attrs = attributes;
  config.numAttrs = 2;
  auto launch = [&](auto chunks) {
    constexpr int kChunks = decltype(chunks)::value;
    constexpr int kMost = kMostChooseWarps;
    return p.keys != nullptr        ? launch_choose<kChunks, kMost, false>(config, p)
           : warps == kMost ? launch_choose<kChunks, kMost, true>(config, p)
                            : launch_choose<kChunks, kMost / 2, true>(config, p);
  };
  switch (p.row) {
    case 64: return launch(std::integral_constant<int, 2>{});
    case 96: return launch(std::integral_constant<int, 3>{});
    case 128: return launch(std::integral_constant<int, 4>{});
    case 192: return launch(std::integral_constant<int, 6>{});
    default: return launch(std::integral_constant<int, 8>{});
  }
}

}  // namespace sb

extern "C" {

int splash_cache_bound(const SplashCacheBoundArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_bound(*args, static_cast<cudaStream_t>(cuda_stream));
}

int splash_cache_bound_values(const SplashKvCache* cache, const SplashPageBounds* bounds, float* values, void* cuda_stream) {
  return cache == nullptr || bounds == nullptr ? SPLASH_ERR_INVALID_ARGUMENT
                                               : sb::cache_bound_values(*cache, *bounds, values, static_cast<cudaStream_t>(cuda_stream));
}

int splash_cache_choose(const SplashCacheChooseArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_choose(*args, static_cast<cudaStream_t>(cuda_stream));
}

size_t splash_cache_choose_workspace_bytes(const SplashCacheChooseArgs* args) { return args == nullptr ? 0 : sb::choose_workspace(*args); }

}  // extern "C"
