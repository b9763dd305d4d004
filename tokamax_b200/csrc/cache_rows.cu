// Rows of the quantised key / value cache: written (quantised) and read back (dequantised).
//
// Both ask for memory alone: a bf16 token row of one head is 256 bytes (head dim 128), its int4 row 64 bytes of codes and
// 8 of scales.  What they come up against first is the number of instructions for a channel, so both keep addresses as
// steps and counters, and their arithmetic short:
//   reading    eight channels a thread (16 bytes on the 16-bit side); bf16 values of four bits by one fused multiply-add in bf16 for
//              two channels.  2 sequences of 16384 tokens, 8 heads of 128, to bf16: 31 us, 5.3 TB/s, from 61 with 32-bit
//              arithmetic and an index per channel; 4 x 32768 from e4m3 120 us, 6.4 TB/s, from 166.
//   writing    sixteen channels a thread; a group's extremes by shuffles between the threads that hold it; quotients by a
//              corrected product.  4 prompts of up to 4096 tokens, bf16 to int4: 27 us, 2.5 TB/s, from 66 with divisions and eight
//              channels a thread; some 340 instructions for sixteen channels, issued at three quarters of the rate that there is.
#include "cache_common.cuh"

namespace sb {

// ------------------------------------------------------------------------------------------
// checks of arguments
// ------------------------------------------------------------------------------------------
static constexpr int kRowWidths[][2] = {{64, 64}, {96, 96}, {128, 128}, {192, 128}, {192, 192}, {256, 256}};

static int row_widths(int head_dim, int head_dim_v, int* row_k, int* row_v) {
  if (head_dim <= 0 || head_dim_v <= 0 || head_dim % 8 != 0 || head_dim_v % 8 != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  for (const auto& w : kRowWidths)
    if (head_dim <= w[0] && head_dim_v <= w[1]) {
      *row_k = w[0];
      *row_v = w[1];
      return SPLASH_OK;
    }
  return SPLASH_ERR_UNSUPPORTED;
}

int check_cache(const SplashKvCache& c) {
  int row_k = 0, row_v = 0;
  if (const int status = row_widths(c.head_dim, c.head_dim_v, &row_k, &row_v)) return status;
  if (c.row_k != row_k || c.row_v != row_v) return SPLASH_ERR_INVALID_ARGUMENT;
  if (c.format != SPLASH_CACHE_INT4 && c.format != SPLASH_CACHE_E4M3) return SPLASH_ERR_UNSUPPORTED;
  if (c.page_size < 16 || (c.page_size & (c.page_size - 1)) != 0 || c.kv_heads <= 0 || c.n_pages <= 0) return SPLASH_ERR_INVALID_ARGUMENT;
  // (rows are counted in 32 bits: more than any GPU holds)
  if (c.n_pages > 0x7fffffffll || c.page_size > (1 << 20) || c.kv_heads > 65535 || c.n_pages > 0xfffffff0ll / c.kv_heads / c.page_size)
    return SPLASH_ERR_TOO_LARGE;
  if (c.format == SPLASH_CACHE_INT4 &&
      ((c.group != 32 && c.group != 64 && c.group != 128) || row_k % c.group != 0 || row_v % c.group != 0))
    return SPLASH_ERR_INVALID_ARGUMENT;
  for (const void* p : {c.k_codes, c.k_scales, c.v_codes, c.v_scales})
    if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u) != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  return SPLASH_OK;
}

int check_cache_tensor(const SplashTensor& t, bool f32_too) {
  if (t.data == nullptr || (reinterpret_cast<uintptr_t>(t.data) & 15u) != 0) return SPLASH_ERR_INVALID_ARGUMENT;
  if (t.dtype != SPLASH_BF16 && t.dtype != SPLASH_F16 && !(f32_too && t.dtype == SPLASH_F32)) return SPLASH_ERR_UNSUPPORTED;
  if (t.stride[3] != 1) return SPLASH_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 4; ++i)
    if (t.size[i] <= 0) return SPLASH_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (t.size[i] > 1 && (t.stride[i] % 8 != 0 || t.stride[i] < 0)) return SPLASH_ERR_INVALID_ARGUMENT;
  return SPLASH_OK;
}

// One side (keys or values) of a cache beside the tensor that is written to it or read from it.
struct RowSide {
  uint8_t* codes;
  uint8_t* scales;
  void* data;
  int64_t stride_b, stride_h, stride_s;
  int32_t head_dim, width;
};

static RowSide side_of(const SplashTensor& t, void* codes, void* scales, int width) {
  return {static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), t.data, t.stride[0], t.stride[1], t.stride[2],
          (int32_t)t.size[3], width};
}

// Calls launch with the threads of a row that have eight channels each: a power of two.
template <typename Fn>
static int with_team(const SplashKvCache& c, Fn&& launch) {
  const int widest = c.row_k > c.row_v ? c.row_k : c.row_v;
  return widest <= 64    ? launch(std::integral_constant<int, 8>{})
         : widest <= 128 ? launch(std::integral_constant<int, 16>{})
                         : launch(std::integral_constant<int, 32>{});
}

// ------------------------------------------------------------------------------------------
// writing
// ------------------------------------------------------------------------------------------
struct AppendParams {
  RowSide side[2];
  const void* slots;
  int64_t slot_stride, n_slots;
  int32_t rows, tokens,  // rows: batch * tokens * kv_heads
      kv_heads, page_size, page_shift, group_shift, slots_are_64;
  uint32_t step_head, step_s, step_b;  // what a row and the next one of a team are apart
};

// With NaN where an operand is NaN (fminf and fmaxf pass the other one on).
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

constexpr int kRowThreads = 256;
constexpr int kWrite = 16;  // channels of a thread that writes

template <int kDType>
struct Loaded {  // sixteen values as they come; of the last eight only what there is
  static constexpr int kWords = kDType == SPLASH_F32 ? 2 : 1;
  uint4 w[2][kWords];
  __device__ __forceinline__ void load(const uint8_t* from, int real) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        w[h][i] = h * 8 < real ? __ldg(reinterpret_cast<const uint4*>(from) + h * kWords + i) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&x)[kWrite]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const uint32_t words[4] = {w[h][i].x, w[h][i].y, w[h][i].z, w[h][i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kDType == SPLASH_F32)
            x[h * 8 + i * 4 + j] = __uint_as_float(words[j]);
          else
            unpack16(kDType, words[j], x[h * 8 + j * 2], x[h * 8 + j * 2 + 1]);
        }
      }
  }
};

// Quantises the channels that a thread has of a row, of which the first `real` (0, 8 or 16) are not padding, and stores them.
// All threads of a warp come along (`kept`: those whose row goes into the cache; the same for all of a row).
template <int kFormat, int kTeam, int kDType>
__device__ __forceinline__ void store_row(const AppendParams& p, const RowSide& side, const float (&x)[kWrite], uint32_t to,
                                          int part, int real, bool kept) {
  if constexpr (kFormat == SPLASH_CACHE_INT4) {
    float least = INFINITY, most = -INFINITY;  // (padding has no part in extremes; its codes are 0)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h * 8 >= real) break;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        least = min_nan(least, x[h * 8 + i], x[h * 8 + i + 1]);
        most = max_nan(most, x[h * 8 + i], x[h * 8 + i + 1]);
      }
    }
    const int threads = 1 << (p.group_shift - 4);  // of a group: 2, 4 or 8, aligned in the warp
    auto exchange = [&](int d) {
      least = min_nan(least, __shfl_xor_sync(~0u, least, d));
      most = max_nan(most, __shfl_xor_sync(~0u, most, d));
    };
    exchange(1);
    if (threads > 2) exchange(2);
    if (threads > 4) exchange(4);
    if (least > most) least = most = 0.f;  // a group of padding alone
    constexpr float kFifteenth = 1.f / 15.f;
    const float range = most - least;
    const __nv_bfloat16 zero_bf = __float2bfloat16_rn(least);
    const __nv_bfloat16 scale_bf = __float2bfloat16_rn(range > kLeastDivisor ? divide(range, 15.f, kFifteenth) : range / 15.f);
    const float zero = __bfloat162float(zero_bf), scale = __bfloat162float(scale_bf);
    const bool finite = range < INFINITY;
    uint32_t codes[2] = {0, 0};
    if (scale > 0.f && finite) {
      const float inverse = __frcp_rn(scale);
      const bool plain = scale <= kLeastDivisor;
      auto quotient = [&](float v) {
        const float d = v - zero, t = plain ? d / scale : divide(d, scale, inverse);
        // (bf16: zero is the least value itself, and a scale of eight bits leaves the quotient within 0 .. 15.06.  A subnormal scale
        // has fewer: 22 for a range of 22 times the least bf16.)
        return kDType == SPLASH_BF16 && !plain ? t : fminf(fmaxf(t, 0.f), 15.f);
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // Rounded to integers by a sum near 2^23 (ties to even), four of them gathered in one number.
        float four[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 3; i >= 0; --i)
#pragma unroll
          for (int j = 0; j < 2; ++j) four[j] = fmaf(four[j], 16.f, (quotient(x[h * 8 + j * 4 + i]) + 8388608.f) - 8388608.f);
        if (h * 8 < real) codes[h] = __byte_perm(__float_as_uint(four[0] + 8388608.f), __float_as_uint(four[1] + 8388608.f), 0x5410);
      }
    }
    if (!kept || part * kWrite >= side.width) return;
    *reinterpret_cast<uint2*>(side.codes + (uint64_t)to * (unsigned)(side.width / 2) + part * 8) = make_uint2(codes[0], codes[1]);
    if ((part & (threads - 1)) == 0) {
      const uint32_t pair = (uint32_t)__bfloat16_as_ushort(zero_bf) | (uint32_t)__bfloat16_as_ushort(scale_bf) << 16;
      const uint64_t row = (uint64_t)to * (unsigned)((side.width >> p.group_shift) * 4);
      *reinterpret_cast<uint32_t*>(side.scales + row + (part * kWrite >> p.group_shift) * 4) = finite ? pair : 0x7fff7fffu;  // NaN, NaN
    }
  } else {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kWrite; i += 2) amax = max_nan(amax, fabsf(x[i]), fabsf(x[i + 1]));
#pragma unroll
    for (int d = 1; d < kTeam; d <<= 1) amax = max_nan(amax, __shfl_xor_sync(~0u, amax, d));
    constexpr float kInverse = 1.f / kE4m3Max;
    const __nv_bfloat16 scale_bf = __float2bfloat16_rn(amax > kLeastDivisor ? divide(amax, kE4m3Max, kInverse) : amax / kE4m3Max);
    const float scale = __bfloat162float(scale_bf);
    const bool finite = amax < INFINITY;
    uint32_t codes[4] = {};
    if (scale > 0.f && finite) {
      const bool plain = scale <= kLeastDivisor;
      const float inverse = __frcp_rn(scale);
#pragma unroll
      for (int i = 0; i < kWrite; i += 2) {
        const float2 t = plain ? make_float2(x[i] / scale, x[i + 1] / scale)
                               : make_float2(divide(x[i], scale, inverse), divide(x[i + 1], scale, inverse));
        codes[i / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3) << (8 * (i % 4));
      }
    }
    if (!kept || part * kWrite >= side.width) return;
    *reinterpret_cast<uint4*>(side.codes + (uint64_t)to * (unsigned)side.width + part * kWrite) =
        make_uint4(codes[0], codes[1], codes[2], codes[3]);
    if (part == 0) reinterpret_cast<uint16_t*>(side.scales)[to] = finite ? __bfloat16_as_ushort(scale_bf) : (uint16_t)0x7fff;
  }
}

// A team of kTeam threads (the power of two that holds the row's width / 16) has a row of one token and head; the rows of a
// token's heads are next to one another, so that the teams of a warp read adjacent memory of a [batch, tokens, heads, d]
// projection.  Teams take rows in turn.  blockIdx.y: keys or values.
template <int kFormat, int kTeam, int kDType>
__global__ void __launch_bounds__(kRowThreads) cache_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kTeams = kRowThreads / kTeam, kBytes = kDType == SPLASH_F32 ? 4 : 2;
  const RowSide& side = p.side[blockIdx.y];
  const int part = threadIdx.x % kTeam;
  const int real = min(max(side.head_dim - part * kWrite, 0), kWrite);
  const unsigned heads = p.kv_heads, tokens = p.tokens, stride = gridDim.x * kTeams;
  unsigned row = blockIdx.x * kTeams + threadIdx.x / kTeam;
  // Where the next row to be looked up stands: token, head; its values' and its slot's addresses.
  unsigned head = row % heads, s = row / heads % tokens;
  const unsigned b = row / heads / tokens;
  const int64_t stride_b = side.stride_b * kBytes, stride_s = side.stride_s * kBytes, stride_h = side.stride_h * kBytes;
  const uint8_t* data = static_cast<const uint8_t*>(side.data) + b * stride_b + s * stride_s + head * stride_h + part * (kWrite * kBytes);
  const int64_t step = p.step_b * stride_b + p.step_s * stride_s + p.step_head * stride_h;
  const int64_t next_token = stride_s - heads * stride_h, next_sequence = stride_b - tokens * stride_s;
  const int slot_bytes = p.slots_are_64 ? 8 : 4;
  const uint8_t* slots = static_cast<const uint8_t*>(p.slots) + (b * p.slot_stride + s) * slot_bytes;
  const int64_t slot_step = (p.step_b * p.slot_stride + p.step_s) * slot_bytes;
  const int64_t slot_next_sequence = (p.slot_stride - (int64_t)tokens) * slot_bytes;
  // A row's values are on their way while the one before it is worked on, its slot a row earlier still: rows that are not kept
  // (padding) are not read.
  constexpr uint32_t kNowhere = ~0u;
  const uint8_t* next_data = nullptr;
  auto look_up = [&]() -> uint32_t {  // where the row goes, in rows of the cache
    uint32_t to = kNowhere;
    next_data = data;
    if (row < (unsigned)p.rows) {
      const int64_t slot =
          p.slots_are_64 ? __ldg(reinterpret_cast<const int64_t*>(slots)) : (int64_t)__ldg(reinterpret_cast<const int32_t*>(slots));
      if (slot >= 0 && slot < p.n_slots)
        to = (((uint32_t)(slot >> p.page_shift) * heads + head) << p.page_shift) + ((uint32_t)slot & (p.page_size - 1));
    }
    row += stride;  // (at most p.rows, below 2^31, and two strides)
    head += p.step_head;
    s += p.step_s;
    data += step;
    slots += slot_step;
    if (head >= heads) {
      head -= heads;
      ++s;
      data += next_token;
      slots += slot_bytes;
    }
    if (s >= tokens) {
      s -= tokens;
      data += next_sequence;
      slots += slot_next_sequence;
    }
    return to;
  };
  uint32_t to = look_up();
  Loaded<kDType> values{};
  if (to != kNowhere) values.load(next_data, real);
  uint32_t next_to = look_up();
  // (whole warps go round together, for their shuffles: as long as the first team of the block has a row)
  for (unsigned row0 = blockIdx.x * kTeams; row0 < (unsigned)p.rows; row0 += stride) {
    float x[kWrite];
    values.get(x);
    const uint32_t now = to;
    to = next_to;
    if (to != kNowhere) values.load(next_data, real);
    next_to = look_up();
    if (__any_sync(~0u, now != kNowhere)) store_row<kFormat, kTeam, kDType>(p, side, x, now, part, real, now != kNowhere);
  }
}

template <int kFormat, int kTeam>
static int launch_append(AppendParams& p, int dtype, cudaStream_t stream) {
  constexpr int kTeams = kRowThreads / kTeam;
  const int64_t blocks = ((int64_t)p.rows + kTeams - 1) / kTeams;
  const dim3 grid((unsigned)(blocks < kSms * 4 ? blocks : kSms * 4), 2);
  const uint32_t stride = grid.x * kTeams, heads = (uint32_t)p.kv_heads, tokens = (uint32_t)p.tokens;
  p.step_head = stride % heads;
  p.step_s = stride / heads % tokens;
  p.step_b = stride / heads / tokens;
  if (dtype == SPLASH_BF16)
    cache_append_kernel<kFormat, kTeam, SPLASH_BF16><<<grid, kRowThreads, 0, stream>>>(p);
  else if (dtype == SPLASH_F16)
    cache_append_kernel<kFormat, kTeam, SPLASH_F16><<<grid, kRowThreads, 0, stream>>>(p);
  else
    cache_append_kernel<kFormat, kTeam, SPLASH_F32><<<grid, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

static int cache_append(const SplashCacheAppendArgs& a, cudaStream_t stream) {
  const SplashKvCache& c = a.cache;
  if (const int status = check_cache(c)) return status;
  for (const SplashTensor* t : {&a.k, &a.v})
    if (const int status = check_cache_tensor(*t, true)) return status;
  if (a.k.dtype != a.v.dtype || a.slots == nullptr || a.slot_stride < 0) return SPLASH_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (a.k.size[i] != a.v.size[i]) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.k.size[1] != c.kv_heads || a.k.size[3] != c.head_dim || a.v.size[3] != c.head_dim_v) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.k.size[0] > 0x7fffffffll || a.k.size[2] > 0x7fffffffll || a.k.size[0] * a.k.size[2] > 0x7fffffffll / c.kv_heads)
    return SPLASH_ERR_TOO_LARGE;
  AppendParams p{};
  p.side[0] = side_of(a.k, c.k_codes, c.k_scales, c.row_k);
  p.side[1] = side_of(a.v, c.v_codes, c.v_scales, c.row_v);
  p.slots = a.slots;
  p.slot_stride = a.slot_stride;
  p.slots_are_64 = a.slots_are_64;
  p.n_slots = c.n_pages * c.page_size;
  p.tokens = (int32_t)a.k.size[2];
  p.kv_heads = c.kv_heads;
  p.rows = (int32_t)(a.k.size[0] * a.k.size[2] * c.kv_heads);
  p.page_size = c.page_size;
  p.page_shift = log2_of(c.page_size);
  p.group_shift = log2_of(c.group);
  return with_team(c, [&](auto team) -> int {
    constexpr int kTeam = decltype(team)::value;
    return c.format == SPLASH_CACHE_INT4 ? launch_append<SPLASH_CACHE_INT4, kTeam / 2>(p, a.k.dtype, stream)
                                         : launch_append<SPLASH_CACHE_E4M3, kTeam / 2>(p, a.k.dtype, stream);
  });
}

// ------------------------------------------------------------------------------------------
// reading
// ------------------------------------------------------------------------------------------
struct ReadParams {
  RowSide side[2];
  const int32_t* page_table;
  const int32_t* lengths;
  int64_t table_stride, n_pages;
  int32_t n_table, max_len, kv_heads, page_size, page_shift, group_shift;
};

constexpr int kReadEach = 8;  // rows of a thread: their loads are in flight together

// a * b + c, rounded to odd: of the two neighbours in 32 bits of a value between them the one whose last bit is 1, which rounds to a
// narrower type as the value itself does (Boldo and Melquiond 2008, "Emulation of FMA and correctly rounded sums: proved
// algorithms using rounding to odd").
__device__ __forceinline__ float fma_odd(float a, float b, float c) {
  const float below = __fmaf_rd(a, b, c), above = __fmaf_ru(a, b, c);
  return __float_as_uint(below) & 1u ? below : above;
}

// zero + scale * code (int4) or scale * code (e4m3, 12 bits) of eight channels, rounded to the type once.
template <int kFormat, int kDType>
__device__ __forceinline__ void store_values(uint8_t* to, uint2 codes, uint32_t scales) {
  if constexpr (kFormat == SPLASH_CACHE_INT4 && kDType == SPLASH_BF16) {
    // Pairs of codes as bf16: 128 + code has the code in its low bits.  The fused multiply-add in bf16 rounds once.
    const uint32_t odd = codes.x >> 4, zero2 = __byte_perm(scales, 0, 0x1010), scale2 = __byte_perm(scales, 0, 0x3232);
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = __byte_perm(codes.x, odd, i | (i + 4) << 8 | i << 4 | (i + 4) << 12) & 0x000f000fu | 0x43004300u;
      asm("{\n\t.reg .b32 c;\n\tadd.rn.bf16x2 c, %1, %4;\n\tfma.rn.bf16x2 %0, c, %2, %3;\n\t}"
          : "=r"(out[i])
          : "r"(w), "r"(scale2), "r"(zero2), "r"(0xc300c300u));
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(out[0], out[1], out[2], out[3]);
  } else {
    const float scale = __uint_as_float(scales & 0xffff0000u), zero = bf16_bits_to_float(scales);
    float x[8];
    if constexpr (kFormat == SPLASH_CACHE_INT4) {
      // (2^23 + code has the code in its low bits: cheaper than a conversion from integers)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(codes.x >> 4 * j & 15u | 0x4b000000u) - 8388608.f;
      // Zero and product are 8 and 12 bits: their sum is one of 32 bits, unless their exponents are far apart.  (f16, 2 x 16384 tokens,
      // 8 heads of 128: 33.8 us without the second form, 39.1 with it alone, 36.3 with both.)
      const int apart = (int)(scales >> 7 & 0xffu) - (int)(scales >> 23 & 0xffu);
      if (kDType == SPLASH_F32 || (apart >= -11 && apart <= 15)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(scale, x[j], zero);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fma_odd(scale, x[j], zero);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = e4m3x2_to_f16x2((j < 2 ? codes.x : codes.y) >> (16 * (j & 1)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        x[2 * j] = scale * f.x;
        x[2 * j + 1] = scale * f.y;
      }
    }
    store8(to, kDType, 0, x);
  }
}

// A team of kTeam threads (as for writing) has a row of one token; a block kReadEach times as many tokens of a (sequence,
// head) as it has teams.  blockIdx.x: tokens, y: head, z: 2 * sequence + (keys or values)
template <int kFormat, int kTeam, int kDType>
__global__ void __launch_bounds__(kRowThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int kTeams = kRowThreads / kTeam, kBytes = kDType == SPLASH_F32 ? 4 : 2;
  const RowSide& side = p.side[blockIdx.z & 1];
  const int b = blockIdx.z >> 1, head = blockIdx.y;
  const int part = threadIdx.x % kTeam;
  if (part * 8 >= side.head_dim) return;
  const int token0 = blockIdx.x * (kTeams * kReadEach) + threadIdx.x / kTeam;  // (below 2^31, as max_len is 2^30 at most)
  const int reach = p.n_table > (p.max_len >> p.page_shift) ? p.max_len : p.n_table << p.page_shift;
  const int length = min(__ldg(p.lengths + b), reach);
  const int32_t* const table = p.page_table + b * p.table_stride;
  int page[kReadEach];
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    const int token = token0 + i * kTeams;
    page[i] = token < length ? __ldg(table + (token >> p.page_shift)) : -1;
  }
  constexpr int kCodeBytes = kFormat == SPLASH_CACHE_INT4 ? 4 : 8;
  const unsigned row_bytes = (unsigned)side.width / 8 * kCodeBytes;
  const unsigned scale_bytes = kFormat == SPLASH_CACHE_INT4 ? (unsigned)(side.width >> p.group_shift) * 4 : 2;
  const uint8_t* const my_codes = side.codes + part * kCodeBytes;
  const uint8_t* const my_scales = side.scales + (kFormat == SPLASH_CACHE_INT4 ? (part * 8 >> p.group_shift) * 4 : 0);
  uint2 codes[kReadEach];
  uint32_t scales[kReadEach];
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    codes[i] = make_uint2(0, 0);
    scales[i] = 0;  // reads as zeros
    if (page[i] < 0 || page[i] >= p.n_pages) continue;
    const uint32_t row = (((uint32_t)page[i] * p.kv_heads + head) << p.page_shift) + ((token0 + i * kTeams) & (p.page_size - 1));
    if constexpr (kFormat == SPLASH_CACHE_INT4) {
      codes[i].x = __ldg(reinterpret_cast<const uint32_t*>(my_codes + (uint64_t)row * row_bytes));
      scales[i] = __ldg(reinterpret_cast<const uint32_t*>(my_scales + (uint64_t)row * scale_bytes));
    } else {
      codes[i] = __ldg(reinterpret_cast<const uint2*>(my_codes + (uint64_t)row * row_bytes));
      scales[i] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(my_scales + (uint64_t)row * scale_bytes)) << 16;
    }
  }
  const int64_t step = side.stride_s * (kTeams * kBytes);
  const int64_t first = b * side.stride_b + head * side.stride_h + token0 * side.stride_s + part * 8;
  uint8_t* to = static_cast<uint8_t*>(side.data) + first * kBytes;
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    if (token0 + i * kTeams < p.max_len) store_values<kFormat, kDType>(to, codes[i], scales[i]);
    to += step;
  }
}

constexpr int64_t kMostSequences = 32767;  // of a launch: two blocks each in a grid's last dimension

template <int kFormat, int kTeam>
static int launch_read(ReadParams p, int dtype, int64_t batch, cudaStream_t stream) {
  constexpr int kTokens = kRowThreads / kTeam * kReadEach;
  for (; batch > 0; batch -= kMostSequences) {
    const int64_t some = batch < kMostSequences ? batch : kMostSequences;
    const dim3 grid((unsigned)((p.max_len + kTokens - 1) / kTokens), (unsigned)p.kv_heads, (unsigned)some * 2);
    if (dtype == SPLASH_BF16)
      cache_read_kernel<kFormat, kTeam, SPLASH_BF16><<<grid, kRowThreads, 0, stream>>>(p);
    else if (dtype == SPLASH_F16)
      cache_read_kernel<kFormat, kTeam, SPLASH_F16><<<grid, kRowThreads, 0, stream>>>(p);
    else
      cache_read_kernel<kFormat, kTeam, SPLASH_F32><<<grid, kRowThreads, 0, stream>>>(p);
    if (cudaGetLastError() != cudaSuccess) return SPLASH_ERR_CUDA;
    p.page_table += some * p.table_stride;
    p.lengths += some;
    for (RowSide& side : p.side) side.data = static_cast<uint8_t*>(side.data) + some * side.stride_b * (dtype == SPLASH_F32 ? 4 : 2);
  }
  return SPLASH_OK;
}

static int cache_read(const SplashCacheReadArgs& a, cudaStream_t stream) {
  const SplashKvCache& c = a.cache;
  if (const int status = check_cache(c)) return status;
  for (const SplashTensor* t : {&a.k, &a.v})
    if (const int status = check_cache_tensor(*t, true)) return status;
  if (a.k.dtype != a.v.dtype || a.page_table == nullptr || a.lengths == nullptr || a.n_table <= 0 || a.table_stride < 0)
    return SPLASH_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (a.k.size[i] != a.v.size[i]) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.k.size[1] != c.kv_heads || a.k.size[3] != c.head_dim || a.v.size[3] != c.head_dim_v) return SPLASH_ERR_INVALID_ARGUMENT;
  if (a.k.size[2] > (1ll << 30) || a.k.size[0] > 0x7fffffffll) return SPLASH_ERR_TOO_LARGE;
  ReadParams p{};
  p.side[0] = side_of(a.k, c.k_codes, c.k_scales, c.row_k);
  p.side[1] = side_of(a.v, c.v_codes, c.v_scales, c.row_v);
  p.page_table = a.page_table;
  p.lengths = a.lengths;
  p.table_stride = a.table_stride;
  p.n_pages = c.n_pages;
  p.n_table = a.n_table;
  p.max_len = (int32_t)a.k.size[2];
  p.kv_heads = c.kv_heads;
  p.page_size = c.page_size;
  p.page_shift = log2_of(c.page_size);
  p.group_shift = log2_of(c.group);
  return with_team(c, [&](auto team) -> int {
    constexpr int kTeam = decltype(team)::value;
    return c.format == SPLASH_CACHE_INT4 ? launch_read<SPLASH_CACHE_INT4, kTeam>(p, a.k.dtype, a.k.size[0], stream)
                                         : launch_read<SPLASH_CACHE_E4M3, kTeam>(p, a.k.dtype, a.k.size[0], stream);
  });
}

}  // namespace sb

extern "C" {

int splash_cache_row_widths(int32_t head_dim, int32_t head_dim_v, int32_t* row_k, int32_t* row_v) {
  return row_k == nullptr || row_v == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::row_widths(head_dim, head_dim_v, row_k, row_v);
}

int splash_cache_append(const SplashCacheAppendArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_append(*args, static_cast<cudaStream_t>(cuda_stream));
}

int splash_cache_read(const SplashCacheReadArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_read(*args, static_cast<cudaStream_t>(cuda_stream));
}

}  // extern "C"
