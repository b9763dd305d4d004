// Which pages of the quantised key / value cache a query attends to: bounds of the keys of whole pages, and the choice of those
// whose bounds allow the largest logits.
//
// Mathematics.  With least_c <= k_c <= largest_c for the keys of a page, q . k <= sum over c of max(q_c least_c, q_c largest_c) =
// sum over c of min(q_c, 0) least_c + max(q_c, 0) largest_c, a product of rows of twice the head dim.  Both sides are held in 8 bits, so
// that the sum is one of whole numbers: it has no rounding, and the choice is the same in any order of summation.  (The 8 bits are
// rounded to the nearest: the sum is a score then, a bound within half a step a channel.)
#include <atomic>

#include "cache_common.cuh"

namespace sb {

constexpr float kMostCode = 127.f;

// NaN as 0 and infinities as the largest number.
__device__ __forceinline__ float as_number(float x) { return x != x ? 0.f : fminf(fmaxf(x, -3.4028234663852886e38f), 3.4028234663852886e38f); }
// round(x / scale) in -127 .. 127
__device__ __forceinline__ int code_of(float x, float scale) {
  return scale > 0.f ? (int)fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -kMostCode), kMostCode) : 0;
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
  int32_t n_table, page_size, page_shift, kv_heads, head_dim, row, group_shift;
};

constexpr int kBoundThreads = 256;

// Eight channels of a row in 32 bits, from its codes and the scales of their group.
template <int kFormat>
struct RowPiece {
  uint32_t w[kFormat == SPLASH_CACHE_INT4 ? 1 : 2];
  uint32_t scale;
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales) {
    if constexpr (kFormat == SPLASH_CACHE_INT4) {
      w[0] = *reinterpret_cast<const uint32_t*>(codes);
      scale = *reinterpret_cast<const uint32_t*>(scales);
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(codes);
      w[0] = v.x, w[1] = v.y;
      scale = (uint32_t)*reinterpret_cast<const uint16_t*>(scales) << 16;
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const float s = __uint_as_float(scale & 0xffff0000u);
    if constexpr (kFormat == SPLASH_CACHE_INT4) {
      const float zero = bf16_bits_to_float(scale);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf(s, __uint_as_float(w[0] >> 4 * j & 15u | 0x4b000000u) - 8388608.f, zero);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = e4m3x2_to_f16x2(w[j / 2] >> (16 * (j & 1)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        x[2 * j] = s * f.x;
        x[2 * j + 1] = s * f.y;
      }
    }
  }
};

// A block has a page of a sequence and kv head: blockIdx.x the page (from the first that has become whole), y the head, z the
// sequence.  A team of row / 8 threads has a token's row, eight channels a thread.
template <int kFormat>
__global__ void __launch_bounds__(kBoundThreads) cache_bound_kernel(const __grid_constant__ BoundParams p) {
  extern __shared__ float extremes[];  // [2][teams][row]
  __shared__ float tops[kBoundThreads / 32];
  const int head = blockIdx.y;
  const int team_size = p.row / 8, teams = kBoundThreads / team_size;
  const int team = threadIdx.x / team_size, part = threadIdx.x % team_size;
  for (int64_t b = blockIdx.z; b < p.batch; b += gridDim.z) {
    const int64_t length = min((int64_t)max(__ldg(p.lengths + b), 0), (int64_t)p.n_table << p.page_shift);
    const int64_t index = (max(length - p.newest, (int64_t)0) >> p.page_shift) + blockIdx.x;
    if (index >= length >> p.page_shift) continue;
    const int page = __ldg(p.page_table + b * p.table_stride + index);
    if (!in_pool(page, p.n_pages)) continue;
    const uint32_t row0 = ((uint32_t)page * p.kv_heads + head) << p.page_shift;
    constexpr int kCodeBytes = kFormat == SPLASH_CACHE_INT4 ? 4 : 8;
    const int row_bytes = team_size * kCodeBytes, scale_bytes = kFormat == SPLASH_CACHE_INT4 ? (p.row >> p.group_shift) * 4 : 2;
    const uint8_t* const codes = p.codes + (uint64_t)row0 * (unsigned)row_bytes + part * kCodeBytes;
    const uint8_t* const scales = p.scales + (uint64_t)row0 * (unsigned)scale_bytes + (kFormat == SPLASH_CACHE_INT4 ? (part * 8 >> p.group_shift) * 4 : 0);
    float least[8], most[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) least[j] = INFINITY, most[j] = -INFINITY;
    if (team < teams) {
#pragma unroll 4
      for (int t = team; t < p.page_size; t += teams) {
        RowPiece<kFormat> piece;
        piece.load(codes + (int64_t)t * row_bytes, scales + (int64_t)t * scale_bytes);
        float x[8];
        piece.get(x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = as_number(x[j]);
          least[j] = fminf(least[j], v);
          most[j] = fmaxf(most[j], v);
        }
      }
      float* const mine = extremes + team * p.row + part * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) mine[j] = least[j], mine[teams * p.row + j] = most[j];
    }
    __syncthreads();
    // a thread a channel (rows are no wider than a block)
    float lo = INFINITY, hi = -INFINITY;
    const bool mine = threadIdx.x < p.head_dim;
    for (int t = 0; mine && t < teams; ++t) {
      lo = fminf(lo, extremes[t * p.row + threadIdx.x]);
      hi = fmaxf(hi, extremes[(teams + t) * p.row + threadIdx.x]);
    }
    float top = mine ? fmaxf(fabsf(lo), fabsf(hi)) : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBoundThreads / 32; ++w) top = fmaxf(top, tops[w]);
    const float scale = __fdiv_rn(top, kMostCode);
    const uint64_t at = (uint64_t)((uint32_t)page * p.kv_heads + head);
    if (threadIdx.x < p.row) {
      int8_t* const to = p.bound_codes + at * (unsigned)(2 * p.row) + threadIdx.x;
      to[0] = (int8_t)(mine ? code_of(lo, scale) : 0);
      to[p.row] = (int8_t)(mine ? code_of(hi, scale) : 0);
    }
    if (threadIdx.x == 0) p.bound_scales[at] = scale;
    __syncthreads();  // (before `extremes` and `tops` are written again)
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
  const dim3 grid((unsigned)(pages < a.n_table ? pages : a.n_table), (unsigned)c.kv_heads, (unsigned)(a.batch < 65535 ? a.batch : 65535));
  const int team = c.row_k / 8, smem = 2 * (kBoundThreads / team) * c.row_k * (int)sizeof(float);  // 16 KB at most
  if (c.format == SPLASH_CACHE_INT4)
    cache_bound_kernel<SPLASH_CACHE_INT4><<<grid, kBoundThreads, smem, stream>>>(p);
  else
    cache_bound_kernel<SPLASH_CACHE_E4M3><<<grid, kBoundThreads, smem, stream>>>(p);
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
  int32_t dtype, batch, kv_heads, heads_per_kv, q_len, n_table, page_size, page_shift, head_dim, row, count, first, last;
};

constexpr int kChooseThreads = 256, kChooseWarps = kChooseThreads / 32;
constexpr int kKeysOnChip = 32768;  // pages of a row whose scores shared memory holds
constexpr int kMostCluster = 8;
constexpr int kBins = 2048, kBinBits = 11;
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

// Shared memory of a CTA: q's codes [heads, to a multiple of 8][2 * row, and 64 bytes], then the keys (of the cluster's first CTA).
__host__ __device__ constexpr int choose_pitch(int row) { return 2 * row + 64; }
__host__ __device__ constexpr int choose_heads(int heads) { return (heads + 7) / 8 * 8; }

struct Found {  // of some of a row's pages
  uint32_t least, most;  // keys but for kAlways
  int candidates, always;
};
__device__ __forceinline__ Found join(Found a, Found b) {
  return {min(a.least, b.least), max(a.most, b.most), a.candidates + b.candidates, a.always + b.always};
}
__device__ __forceinline__ Found join_warp(Found f) {
  return {__reduce_min_sync(~0u, f.least), __reduce_max_sync(~0u, f.most), __reduce_add_sync(~0u, f.candidates), __reduce_add_sync(~0u, f.always)};
}

// Sum over the threads of a CTA before this one; `total` of all.  One word of `scratch` a warp.
__device__ __forceinline__ uint64_t sum_before(uint64_t mine, uint64_t* scratch, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t other = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += other;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  uint64_t before = sum - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < kChooseWarps; ++w) {
    before += w < warp ? scratch[w] : 0;
    total += scratch[w];
  }
  __syncthreads();
  return before;
}

// A cluster (of one CTA and more) has a query and kv head: its CTAs score pages, tile by tile of 16, and the first one chooses.
__global__ void __launch_bounds__(kChooseThreads) cache_choose_kernel(const __grid_constant__ ChooseParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t scratch[kChooseWarps];
  __shared__ Found parts[kMostCluster * kChooseWarps];
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t found_bin[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  uint32_t ctas, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const uint32_t row = blockIdx.x / ctas;  // (sequence, kv head, query)
  const int i = row % (unsigned)p.q_len, head = row / (unsigned)p.q_len % (unsigned)p.kv_heads, b = row / (unsigned)p.q_len / (unsigned)p.kv_heads;
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  const int64_t reach = (int64_t)p.n_table << p.page_shift;
  const int position = (int)min(max((int64_t)__ldg(p.lengths + b) - p.q_len + i, (int64_t)-1), reach - 1);
  const int own = position >> p.page_shift, pages = own + 1;  // (-1 and 0 before the sequence)

  // ---- q in 8 bits ----
  const int vectors = p.head_dim / 8, pitch = choose_pitch(p.row);
  const uint16_t* const q = static_cast<const uint16_t*>(p.q) + b * p.q_stride_b + (int64_t)head * p.heads_per_kv * p.q_stride_h + i * p.q_stride_s;
  auto load_q = [&](int at, float (&x)[8]) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q + at / vectors * p.q_stride_h + at % vectors * 8));
    unpack16(p.dtype, w.x, x[0], x[1]);
    unpack16(p.dtype, w.y, x[2], x[3]);
    unpack16(p.dtype, w.z, x[4], x[5]);
    unpack16(p.dtype, w.w, x[6], x[7]);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = as_number(x[k]);
  };
  float x[8] = {}, top = 0.f;
  for (int at = tid; at < vectors * p.heads_per_kv; at += kChooseThreads) {
    load_q(at, x);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[k]));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  float* const tops = reinterpret_cast<float*>(scratch);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kChooseWarps; ++w) top = fmaxf(top, tops[w]);
  const float scale = __fdiv_rn(top, kMostCode);
  const int heads = choose_heads(p.heads_per_kv), row_vectors = p.row / 8;
  for (int at = tid; at < heads * row_vectors; at += kChooseThreads) {
    const int h = at / row_vectors, d = at % row_vectors;
    uint32_t negative[2] = {0, 0}, positive[2] = {0, 0};
    if (d < vectors) {
      load_q((h < p.heads_per_kv ? h : 0) * vectors + d, x);  // (rows that make up eight repeat the first one)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int code = code_of(x[k], scale);
        negative[k / 4] |= (uint32_t)(min(code, 0) & 255) << 8 * (k % 4);
        positive[k / 4] |= (uint32_t)max(code, 0) << 8 * (k % 4);
      }
    }
    *reinterpret_cast<uint2*>(smem + h * pitch + d * 8) = make_uint2(negative[0], negative[1]);
    *reinterpret_cast<uint2*>(smem + h * pitch + p.row + d * 8) = make_uint2(positive[0], positive[1]);
  }
  __syncthreads();

  // ---- scores ----
  uint32_t* const own_keys = p.keys != nullptr ? p.keys + (uint64_t)row * p.n_table : reinterpret_cast<uint32_t*>(smem + heads * pitch);
  uint32_t* to_keys = own_keys;
  Found* to_parts = parts;
  if (ctas > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // (the first CTA is there)
    uint64_t at;
    if (p.keys == nullptr) {
      asm("mapa.u64 %0, %1, 0;" : "=l"(at) : "l"(reinterpret_cast<uint64_t>(own_keys)));
      to_keys = reinterpret_cast<uint32_t*>(at);
    }
    asm("mapa.u64 %0, %1, 0;" : "=l"(at) : "l"(reinterpret_cast<uint64_t>(to_parts)));
    to_parts = reinterpret_cast<Found*>(at);
  }
  Found found{~0u, 0u, 0, 0};
  const int32_t* const table = p.page_table + b * p.table_stride;
  const int step = (int)ctas * kChooseWarps * 16, chunks = p.row / 32;
  auto look_up = [&](int index) {
    const int page = index < pages ? __ldg(table + index) : -1;
    return in_pool(page, p.n_pages) ? page : -1;
  };
  int first = ((int)rank + warp * (int)ctas) * 16;
  int page0 = look_up(first + g), page1 = look_up(first + 8 + g);
  for (; first < pages; first += step) {
    const int next0 = look_up(first + step + g), next1 = look_up(first + step + 8 + g);
    // (pages that are no candidates are read as page 0)
    const uint64_t at0 = (uint64_t)max(page0, 0) * p.kv_heads + head, at1 = (uint64_t)max(page1, 0) * p.kv_heads + head;
    const uint4* const from0 = reinterpret_cast<const uint4*>(p.bound_codes + at0 * (unsigned)(2 * p.row)) + t4;
    const uint4* const from1 = reinterpret_cast<const uint4*>(p.bound_codes + at1 * (unsigned)(2 * p.row)) + t4;
    const int mine = t4 & 1;  // lanes 0 and 1 of four have a page each
    const float page_scale = __ldg(p.bound_scales + (mine ? at1 : at0));
    int best0 = INT32_MIN, best1 = INT32_MIN;
    for (int h0 = 0; h0 < heads; h0 += 8) {
      const uint8_t* const codes = smem + (h0 + g) * pitch + t4 * 16;
      int c[4] = {};
#pragma unroll 4
      for (int k = 0; k < chunks; ++k) {
        const uint4 a = __ldg(from0 + k * 4), a8 = __ldg(from1 + k * 4);
        const uint4 w = *reinterpret_cast<const uint4*>(codes + k * 64);
        mma_s8(c, a.x, a8.x, a.y, a8.y, w.x, w.y);
        mma_s8(c, a.z, a8.z, a.w, a8.w, w.z, w.w);
      }
      best0 = max(best0, max(c[0], c[1]));
      best1 = max(best1, max(c[2], c[3]));
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      best0 = max(best0, __shfl_xor_sync(~0u, best0, d));
      best1 = max(best1, __shfl_xor_sync(~0u, best1, d));
    }
    const int index = first + mine * 8 + g;
    if (t4 < 2 && index < pages) {
      uint32_t key = key_of((float)(mine ? best1 : best0) * page_scale);
      if ((mine ? page1 : page0) < 0)
        key = kNoCandidate;
      else if (index < p.first || index > own - p.last)
        key = kAlways;
      to_keys[index] = key;
      found.candidates += key != kNoCandidate;
      found.always += key == kAlways;
      if (key != kNoCandidate && key != kAlways) {
        found.least = min(found.least, key);
        found.most = max(found.most, key);
      }
    }
    page0 = next0;
    page1 = next1;
  }
  __syncwarp();
  found = join_warp(found);
  if (lane == 0) to_parts[rank * kChooseWarps + warp] = found;
  __syncwarp();
  if (ctas > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // ---- the least key that is taken, and how many of those equal to it ----
  found = {~0u, 0u, 0, 0};
  for (int w = lane; w < (int)ctas * kChooseWarps; w += 32) found = join(found, parts[w]);
  found = join_warp(found);
  uint32_t threshold = 1;  // all candidates
  int wanted = p.count, equal = INT32_MAX;
  if (found.candidates > wanted) {
    wanted -= found.always;  // of the others; fewer than there are
    // Digits of key - least, from the highest: of each the bin that the wanted-th largest key lies in.
    const uint32_t range = found.most - found.least;
    int bits = 32 - __clz(range);  // of the differences
    uint32_t prefix = 0;           // of the difference, above `bits`
    threshold = kAlways;
    equal = 0;
    while (wanted > 0) {
      const int shift = max(bits - kBinBits, 0);
      for (int k = tid; k < kBins; k += kChooseThreads) bins[k] = 0;
      __syncthreads();
      for (int k = tid; k < pages; k += kChooseThreads) {
        const uint32_t key = own_keys[k], difference = key - found.least;
        if (key != kNoCandidate && key != kAlways && (bits == 32 ? 0 : difference >> bits) == prefix)
          atomicAdd(&bins[difference >> shift & ((1u << (bits - shift)) - 1)], 1u);
      }
      __syncthreads();
      // bins from the highest: a thread has kBins / kChooseThreads of them
      constexpr int kEach = kBins / kChooseThreads;
      uint32_t own_bins[kEach], sum = 0;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        own_bins[k] = bins[kBins - 1 - (tid * kEach + k)];
        sum += own_bins[k];
      }
      uint64_t total;
      uint32_t before = (uint32_t)sum_before(sum, scratch, total);
      if (before < (uint32_t)wanted && before + sum >= (uint32_t)wanted) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          if (before < (uint32_t)wanted && before + own_bins[k] >= (uint32_t)wanted) {
            found_bin[0] = kBins - 1 - (tid * kEach + k);
            found_bin[1] = before;
          }
          before += own_bins[k];
        }
      }
      __syncthreads();
      prefix = prefix << (bits - shift) | found_bin[0];
      wanted -= (int)found_bin[1];
      bits = shift;
      if (bits == 0) {
        threshold = found.least + prefix;
        equal = wanted;
        break;
      }
      __syncthreads();  // (before bins and found_bin are written again)
    }
  }

  // ---- the pages taken, in order: a thread has a run of them ----
  const int run = (pages + kChooseThreads - 1) / kChooseThreads, from = min(tid * run, pages), until = min(from + run, pages);
  uint64_t counts = 0;  // taken whatever comes, and equal to the threshold
  for (int k = from; k < until; ++k) {
    const uint32_t key = own_keys[k];
    counts += (key > threshold || key == kAlways ? 1ull : 0ull) | (key == threshold && key != kAlways ? 1ull << 32 : 0ull);
  }
  uint64_t total;
  const uint64_t before = sum_before(counts, scratch, total);
  int equals = (int)(before >> 32), taken = (int)(uint32_t)before + min(equals, equal);
  int32_t* const to = p.tables + (uint64_t)row * p.count;
  for (int k = from; k < until; ++k) {
    const uint32_t key = own_keys[k];
    bool take = key > threshold || key == kAlways;
    if (key == threshold && key != kAlways) take = equals++ < equal;
    if (take) to[taken++] = __ldg(table + k);
  }
  const int all = (int)(uint32_t)total + min((int)(total >> 32), equal);
  for (int k = all + tid; k < p.count; k += kChooseThreads) to[k] = -1;
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
      (int64_t)a.count * c.page_size > (1 << 30) || a.q.size[1] / c.kv_heads > 128)
    return SPLASH_ERR_TOO_LARGE;
  return SPLASH_OK;
}

static size_t choose_workspace(const SplashCacheChooseArgs& a) {
  if (check_choose(a) != SPLASH_OK || a.n_table <= kKeysOnChip) return 0;
  return (size_t)(a.q.size[0] * a.cache.kv_heads * a.q.size[2]) * a.n_table * sizeof(uint32_t);
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
  p.batch = (int32_t)a.q.size[0];
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
  int ctas = 1;
  while (ctas < kMostCluster && rows * ctas * 2 <= 2 * kSms && (int64_t)a.n_table > (int64_t)ctas * kChooseWarps * 16) ctas *= 2;
  const int smem = choose_heads(p.heads_per_kv) * choose_pitch(p.row) + (p.keys == nullptr ? a.n_table * 4 : 0);
  static std::atomic<uint64_t> ready{0};  // devices that know how much shared memory the kernel takes
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return SPLASH_ERR_CUDA;
  const uint64_t bit = 1ull << (device & 63);
  constexpr int kMostShared = 128 * choose_pitch(256) + kKeysOnChip * 4;
  static_assert(kMostShared + 12 * 1024 <= 227 * 1024);
  if (device > 63 || !(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(cache_choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return SPLASH_ERR_CUDA;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(rows * ctas));
  config.blockDim = dim3(kChooseThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = ctas;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, cache_choose_kernel, p) == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

}  // namespace sb

extern "C" {

int splash_cache_bound(const SplashCacheBoundArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_bound(*args, static_cast<cudaStream_t>(cuda_stream));
}

int splash_cache_choose(const SplashCacheChooseArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::cache_choose(*args, static_cast<cudaStream_t>(cuda_stream));
}

size_t splash_cache_choose_workspace_bytes(const SplashCacheChooseArgs* args) { return args == nullptr ? 0 : sb::choose_workspace(*args); }

}  // extern "C"
