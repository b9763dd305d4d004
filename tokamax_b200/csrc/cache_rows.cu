// Rows of the quantised key / value cache: written (quantised) and read back (dequantised).
//
// Both are bound by memory: a bf16 token row of one head is 256 bytes (head dim 128), its int4 row 64 bytes of codes and
// 8 of scales.  A thread holds eight channels, 16 bytes on the 16-bit side and 4 (int4) or 8 (e4m3) on the cache's; a
// group's extremes come from shuffles between the threads that hold it.
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
  if (c.n_pages > 0x7fffffffll || c.page_size > (1 << 20) || c.kv_heads > 65535) return SPLASH_ERR_TOO_LARGE;
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

// ------------------------------------------------------------------------------------------
// writing
// ------------------------------------------------------------------------------------------
struct AppendParams {
  RowSide side[2];
  const void* slots;
  int64_t slot_stride, n_slots;
  int32_t rows, tokens,  // rows: batch * tokens * kv_heads
       kv_heads, page_size, page_shift, group, dtype, slots_are_64;
};

// A team of `kTeam` threads (the power of two that holds the row's width / 8) has one row of one token and head; rows
// of a token's heads are next to one another, so that the teams of a warp read adjacent memory of a [batch, tokens,
// heads, d] projection.
template <int kFormat, int kTeam>
__device__ __forceinline__ void append_row(const AppendParams& p, const RowSide& side, int row, int part) {
  const unsigned token = (unsigned)row / (unsigned)p.kv_heads, head = (unsigned)row % (unsigned)p.kv_heads;
  const int64_t b = token / (unsigned)p.tokens, s = token % (unsigned)p.tokens;
  const int64_t at = b * p.slot_stride + s;
  const int64_t slot = p.slots_are_64 ? __ldg(static_cast<const int64_t*>(p.slots) + at) : (int64_t)__ldg(static_cast<const int32_t*>(p.slots) + at);
  const bool kept = slot >= 0 && slot < p.n_slots;  // (the same for the whole team)
  const bool real = part * 8 < side.head_dim;       // (padding beyond it has no part in extremes; its codes are 0)
  float x[8] = {};
  if (kept && real) load8(side.data, p.dtype, b * side.stride_b + head * side.stride_h + s * side.stride_s + part * 8, x);
  const int64_t page = slot >> p.page_shift;
  const int64_t to = (page * p.kv_heads + head) * p.page_size + (slot & (p.page_size - 1));

  if constexpr (kFormat == SPLASH_CACHE_INT4) {
    float least = INFINITY, most = -INFINITY;
    bool finite = true;
    if (real) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        least = fminf(least, x[i]);
        most = fmaxf(most, x[i]);
        finite = finite && fabsf(x[i]) < INFINITY;  // (not for NaN either)
      }
    }
    const int threads = p.group / 8;  // of a group: 4, 8 or 16, aligned in the warp
    for (int d = 1; d < threads; d <<= 1) {  // (a group that is partly padding has its extremes from the rest)
      least = fminf(least, __shfl_xor_sync(~0u, least, d));
      most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
      finite = __shfl_xor_sync(~0u, finite, d) && finite;
    }
    if (!(least <= most)) least = most = 0.f;  // a group of padding alone
    const __nv_bfloat16 zero_bf = __float2bfloat16_rn(least), scale_bf = __float2bfloat16_rn((most - least) / 15.0f);
    const float zero = __bfloat162float(zero_bf), scale = __bfloat162float(scale_bf);
    uint32_t codes = 0;
    if (real && scale > 0.f && finite) {
#pragma unroll
      for (int i = 0; i < 8; ++i) codes |= (uint32_t)fminf(fmaxf(rintf((x[i] - zero) / scale), 0.f), 15.f) << (4 * i);
    }
    if (!kept || part * 8 >= side.width) return;
    const int row_words = side.width / 8;
    reinterpret_cast<uint32_t*>(side.codes)[to * row_words + part] = codes;
    if ((part & (threads - 1)) == 0) {
      uint32_t pair = (uint32_t)__bfloat16_as_ushort(zero_bf) | (uint32_t)__bfloat16_as_ushort(scale_bf) << 16;
      if (!finite) pair = 0x7fff7fffu;  // NaN, NaN
      reinterpret_cast<uint32_t*>(side.scales)[to * (side.width / p.group) + part / threads] = pair;
    }
  } else {
    float amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      amax = fmaxf(amax, fabsf(x[i]));
      finite = finite && fabsf(x[i]) < INFINITY;
    }
#pragma unroll
    for (int d = 1; d < kTeam; d <<= 1) {
      amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, d));
      finite = __shfl_xor_sync(~0u, finite, d) && finite;
    }
    const __nv_bfloat16 scale_bf = __float2bfloat16_rn(amax / kE4m3Max);
    const float scale = __bfloat162float(scale_bf);
    uint32_t codes[2] = {0, 0};
    if (scale > 0.f && finite) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        codes[i / 4] |= (uint32_t)__nv_cvt_float_to_fp8(x[i] / scale, __NV_SATFINITE, __NV_E4M3) << (8 * (i % 4));
    }
    if (!kept || part * 8 >= side.width) return;
    reinterpret_cast<uint2*>(side.codes)[to * (side.width / 8) + part] = make_uint2(codes[0], codes[1]);
    if (part == 0) reinterpret_cast<uint16_t*>(side.scales)[to] = finite ? __bfloat16_as_ushort(scale_bf) : (uint16_t)0x7fff;
  }
}

constexpr int kRowThreads = 256;

// blockIdx.y: keys or values
template <int kFormat, int kTeam>
__global__ void __launch_bounds__(kRowThreads) cache_append_kernel(const __grid_constant__ AppendParams p) {
  const int64_t id = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const int64_t row = id / kTeam;
  const bool inside = row < p.rows;
  // (threads behind the last row go along, for the shuffles, on a row that they do not store)
  append_row<kFormat, kTeam>(p, p.side[blockIdx.y], inside ? (int)row : p.rows - 1, inside ? (int)(id % kTeam) : kTeam * 8);
}

template <int kFormat>
static int launch_append(const AppendParams& p, int team, cudaStream_t stream) {
  const int64_t blocks = ((int64_t)p.rows * team + kRowThreads - 1) / kRowThreads;
  const dim3 grid((unsigned)blocks, 2);
  if (team == 8)
    cache_append_kernel<kFormat, 8><<<grid, kRowThreads, 0, stream>>>(p);
  else if (team == 16)
    cache_append_kernel<kFormat, 16><<<grid, kRowThreads, 0, stream>>>(p);
  else
    cache_append_kernel<kFormat, 32><<<grid, kRowThreads, 0, stream>>>(p);
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
  p.group = c.group;
  p.dtype = a.k.dtype;
  const int widest = c.row_k > c.row_v ? c.row_k : c.row_v;
  const int team = widest <= 64 ? 8 : widest <= 128 ? 16 : 32;
  return c.format == SPLASH_CACHE_INT4 ? launch_append<SPLASH_CACHE_INT4>(p, team, stream)
                                       : launch_append<SPLASH_CACHE_E4M3>(p, team, stream);
}

// ------------------------------------------------------------------------------------------
// reading
// ------------------------------------------------------------------------------------------
struct ReadParams {
  RowSide side[2];
  const int32_t* page_table;
  const int32_t* lengths;
  int64_t table_stride, n_pages;
  int32_t n_table, max_len, kv_heads, page_size, page_shift, group, dtype;
};

constexpr int kReadEach = 4;  // pieces of eight channels a thread: their loads are in flight together

// blockIdx.x: pieces of a (sequence, head), z: 2 * sequence + (keys or values), y: head
template <int kFormat>
__global__ void __launch_bounds__(kRowThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
  const RowSide& side = p.side[blockIdx.z & 1];
  const int b = blockIdx.z >> 1, head = blockIdx.y;
  const int pieces = side.head_dim / 8;  // of a row
  const int length = min(__ldg(p.lengths + b), p.max_len);
  const int64_t first = (int64_t)blockIdx.x * (kRowThreads * kReadEach) + threadIdx.x;
  int token[kReadEach], part[kReadEach];
  uint2 codes[kReadEach];
  uint32_t scales[kReadEach];
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    const int64_t id = first + i * kRowThreads;
    token[i] = id < (int64_t)p.max_len * pieces ? (int)((uint64_t)id / (unsigned)pieces) : -1;
    part[i] = (int)(id - (int64_t)token[i] * pieces);
    codes[i] = make_uint2(0, 0);
    scales[i] = 0;  // reads as zeros
    if (token[i] < 0 || token[i] >= length) continue;
    const int at = token[i] >> p.page_shift;
    const int page = at < p.n_table ? __ldg(p.page_table + b * p.table_stride + at) : -1;
    if (page < 0 || page >= p.n_pages) continue;
    const int64_t row = ((int64_t)page * p.kv_heads + head) * p.page_size + (token[i] & (p.page_size - 1));
    if (kFormat == SPLASH_CACHE_INT4) {
      codes[i].x = __ldg(reinterpret_cast<const uint32_t*>(side.codes) + row * (side.width / 8) + part[i]);
      scales[i] = __ldg(reinterpret_cast<const uint32_t*>(side.scales) + row * (side.width / p.group) + part[i] * 8 / p.group);
    } else {
      codes[i] = __ldg(reinterpret_cast<const uint2*>(side.codes) + row * (side.width / 8) + part[i]);
      scales[i] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(side.scales) + row) << 16;
    }
  }
#pragma unroll
  for (int i = 0; i < kReadEach; ++i) {
    if (token[i] < 0) continue;
    const float scale = __uint_as_float(scales[i] & 0xffff0000u), zero = bf16_bits_to_float(scales[i]);
    float x[8];
    if (kFormat == SPLASH_CACHE_INT4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf(scale, (float)((codes[i].x >> (4 * j)) & 15u), zero);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = e4m3x2_to_f16x2((j < 2 ? codes[i].x : codes[i].y) >> (16 * (j & 1)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        x[2 * j] = scale * f.x;
        x[2 * j + 1] = scale * f.y;
      }
    }
    store8(side.data, p.dtype, b * side.stride_b + head * side.stride_h + token[i] * side.stride_s + part[i] * 8, x);
  }
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
  if (a.k.size[2] > 0x7fffffffll || a.k.size[0] > 32767) return SPLASH_ERR_TOO_LARGE;
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
  p.group = c.group;
  p.dtype = a.k.dtype;
  const int wider = c.head_dim > c.head_dim_v ? c.head_dim : c.head_dim_v;
  const int64_t per_block = kRowThreads * kReadEach;
  const int64_t blocks = (a.k.size[2] * (wider / 8) + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return SPLASH_ERR_TOO_LARGE;
  const dim3 grid((unsigned)blocks, (unsigned)c.kv_heads, (unsigned)a.k.size[0] * 2);
  if (c.format == SPLASH_CACHE_INT4)
    cache_read_kernel<SPLASH_CACHE_INT4><<<grid, kRowThreads, 0, stream>>>(p);
  else
    cache_read_kernel<SPLASH_CACHE_E4M3><<<grid, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
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
