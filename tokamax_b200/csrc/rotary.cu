// Rotary positions of queries and keys, and their gradient.
//
// Mathematics.  Pair i of a row's first channels, as a complex number, times factor * exp(2 pi I * position * turns[i]); the gradient is
// the product with the conjugate.  Angles are fixed-point fractions of a whole turn, 64 bits: position * turns modulo 2^64 drops
// whole turns exactly, at any position, with one integer multiplication, where a product in floating point loses the
// fraction of a turn as positions grow (32 bits: 0.06 radians at 10^6).  The 32 high bits go to sincospi as half turns, in 24 bits: up to
// 2^-25 of a half turn off, 1e-7 of a pair, which rows of 16 bits do not see.  For rows of 32 bits whole quarters of a turn are taken off first:
// what is left has 24 bits of its own, and sine and cosine are right to their last places at any angle.
//
// Bound by memory: a value is read once and written once.  A thread has the same eight pairs of a token for four heads: an angle, its
// sine and cosine are worked out once for them, and eight loads of 16 bytes are in flight.  4 x 4096 tokens, 32 + 8 heads of 128, bf16:
// 54.8 us, 6.1 TB/s (a plain copy of the same tensors 58.4, each input and output once at the copy rate 51.3); with two heads a
// thread 70, with ten 59.6, forty 66.6; eight loads ahead 74.  2 x 8192 forward and back 104.7 (floor 102.6).  Interleaved 55.0.  f32 105.5 (floor
// 102.6), interleaved 125.  80 channels, bf16 (floor 32.1): all of them turned 37.3; 72 or 40, whose pairs come in fours, 40; 20, whose pairs go one
// by one, two bytes a load, 101.
// Evicting loads and stores, and blocks of 128, +-1 %.
#include "cache_common.cuh"

namespace sb {

struct RotateSide {
  const uint8_t* x;
  uint8_t* y;
  int64_t x_b, x_h, x_s, y_b, y_h, y_s;  // strides, bytes
  int32_t heads;
};

struct RotateParams {
  RotateSide side[2];
  const void* positions;
  const uint64_t* turns;
  int64_t position_stride;
  uint32_t rows, tokens;  // rows: batch * tokens
  int32_t head_dim, dim, lanes, rows_each, heads_each, positions_are_64;
  float factor, sign;
};

constexpr int kRotateThreads = 256, kRotateAhead = 4;

// kCount consecutive values of a type, as they lie in memory.
template <int kDType, int kCount>
struct Values {
  static constexpr int kSize = kDType == SPLASH_F32 ? 4 : 2, kBytes = kCount * kSize, kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const uint8_t* from) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(from + i * 4);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(from);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(from);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(from);
    }
  }
  __device__ __forceinline__ void store(uint8_t* to) const {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(to + i * 4) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(to) = w[0];
    } else {
      *reinterpret_cast<uint16_t*>(to) = (uint16_t)w[0];
    }
  }
  __device__ __forceinline__ void get(float (&f)[kCount]) const {
    if constexpr (kDType == SPLASH_F32) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        float lo, hi;
        unpack16(kDType, w[i], lo, hi);
        f[2 * i] = lo;
        if (kCount > 1) f[2 * i + (kCount > 1)] = hi;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[kCount]) {
    if constexpr (kDType == SPLASH_F32) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = pack16(kDType, f[2 * i], kCount > 1 ? f[2 * i + (kCount > 1)] : 0.f);
    }
  }
};

// A lane of a row has 2 * kPairs channels: kPairs pairs, or as many channels that are copied.  `lanes` threads have a row, a block
// rows_each rows; blockIdx.y: the heads.
template <int kDType, int kPairs, bool kInterleaved>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(const __grid_constant__ RotateParams p) {
  using V = Values<kDType, kPairs>;
  const int lane = threadIdx.x % p.lanes;
  const uint32_t row = blockIdx.x * (uint32_t)p.rows_each + threadIdx.x / p.lanes;
  if (row >= p.rows) return;
  const uint32_t b = row / p.tokens, s = row - b * p.tokens;
  const int turned_lanes = p.dim / (2 * kPairs);
  const bool turned = lane < turned_lanes;
  // the channels of a lane: kPairs from c0 on, and from c1 on
  const int c0 = turned ? lane * (kInterleaved ? 2 * kPairs : kPairs) : p.dim + (lane - turned_lanes) * 2 * kPairs;
  const int c1 = turned && !kInterleaved ? c0 + p.dim / 2 : c0 + kPairs;
  const bool both = c1 < p.head_dim;
  float cosine[kPairs], sine[kPairs];
  if (turned) {
    const int64_t at = b * p.position_stride + s;
    const uint64_t position = (uint64_t)(p.positions_are_64 ? __ldg(static_cast<const int64_t*>(p.positions) + at)
                                                            : (int64_t)__ldg(static_cast<const int32_t*>(p.positions) + at));
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t angle = (uint32_t)(position * __ldg(p.turns + lane * kPairs + i) >> 32);  // 2^-31 of a half turn
      if constexpr (kDType == SPLASH_F32) {
        const uint32_t quarters = (angle + 0x20000000u) >> 30;  // (to the nearest)
        float s, c;
        sincospif((float)(int32_t)(angle - (quarters << 30)) * 0x1p-31f, &s, &c);
        sine[i] = quarters & 1 ? c : s;
        cosine[i] = quarters & 1 ? s : c;
        if (quarters & 2) sine[i] = -sine[i];
        if ((quarters + 1) & 2) cosine[i] = -cosine[i];
      } else {
        sincospif((float)(int32_t)angle * 0x1p-31f, &sine[i], &cosine[i]);
      }
      sine[i] *= p.factor * p.sign;
      cosine[i] *= p.factor;
    }
  }
  const int h0 = blockIdx.y * p.heads_each, h1 = min(h0 + p.heads_each, p.side[0].heads + p.side[1].heads);
  auto from = [&](int h) {
    const int which = h >= p.side[0].heads;
    const RotateSide& side = p.side[which];
    return side.x + b * side.x_b + s * side.x_s + (which ? h - p.side[0].heads : h) * side.x_h;
  };
  auto to = [&](int h) {
    const int which = h >= p.side[0].heads;
    const RotateSide& side = p.side[which];
    return side.y + b * side.y_b + s * side.y_s + (which ? h - p.side[0].heads : h) * side.y_h;
  };
  for (int h = h0; h < h1; h += kRotateAhead) {
    V one[kRotateAhead], two[kRotateAhead];
#pragma unroll
    for (int i = 0; i < kRotateAhead; ++i) {
      if (h + i >= h1) break;
      const uint8_t* const x = from(h + i);
      one[i].load(x + c0 * V::kSize);
      if (both) two[i].load(x + c1 * V::kSize);
    }
#pragma unroll
    for (int i = 0; i < kRotateAhead; ++i) {
      if (h + i >= h1) break;
      if (turned) {
        float u[kPairs], v[kPairs], a[kPairs], c[kPairs];
        one[i].get(u);
        two[i].get(v);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          if constexpr (kInterleaved && kPairs > 1) {
            // pairs of neighbours: the first half of them in u, the second in v
            const float (&x)[kPairs] = 2 * j < kPairs ? u : v;
            float (&y)[kPairs] = 2 * j < kPairs ? a : c;
            const int k = 2 * j % kPairs;
            y[k] = x[k] * cosine[j] - x[k + 1] * sine[j];
            y[k + 1] = x[k + 1] * cosine[j] + x[k] * sine[j];
          } else {
            a[j] = u[j] * cosine[j] - v[j] * sine[j];
            c[j] = v[j] * cosine[j] + u[j] * sine[j];
          }
        }
        one[i].set(a);
        two[i].set(c);
      }
      uint8_t* const y = to(h + i);
      one[i].store(y + c0 * V::kSize);
      if (both) two[i].store(y + c1 * V::kSize);
    }
  }
}

template <int kDType, int kPairs>
static int launch_rotate(RotateParams& p, bool interleaved, cudaStream_t stream) {
  p.lanes = p.dim / (2 * kPairs) + (p.head_dim - p.dim + 2 * kPairs - 1) / (2 * kPairs);
  p.rows_each = kRotateThreads / p.lanes;
  const int heads = p.side[0].heads + p.side[1].heads;
  // Four heads a thread, whose loads are in flight together, unless that leaves the GPU without threads.
  p.heads_each = (int64_t)p.rows * p.lanes * heads < (int64_t)kSms * 2048 && heads <= 65535 ? 1 : kRotateAhead;
  const dim3 grid((p.rows + p.rows_each - 1) / p.rows_each, (unsigned)((heads + p.heads_each - 1) / p.heads_each));
  const int block = p.rows_each * p.lanes;
  if (interleaved)
    rotate_kernel<kDType, kPairs, true><<<grid, block, 0, stream>>>(p);
  else
    rotate_kernel<kDType, kPairs, false><<<grid, block, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? SPLASH_OK : SPLASH_ERR_CUDA;
}

template <int kDType>
static int pick_rotate(RotateParams& p, bool interleaved, cudaStream_t stream) {
  // Eight pairs a lane, 16 bytes of a 16-bit type, where the pairs come in eights, else four or one (two bytes at a time: for widths
  // such as 20 of 80 channels, which have no better alignment).
  if (p.dim % 16 == 0) return launch_rotate<kDType, 8>(p, interleaved, stream);
  if (p.dim % 8 == 0) return launch_rotate<kDType, 4>(p, interleaved, stream);
  return launch_rotate<kDType, 1>(p, interleaved, stream);
}

static int rotate(const SplashRotateArgs& a, cudaStream_t stream) {
  RotateParams p{};
  const SplashTensor* shape = nullptr;
  for (int i = 0; i < 2; ++i) {
    const SplashTensor &x = a.x[i], &y = a.y[i];
    if (x.data == nullptr && y.data == nullptr) continue;
    for (const SplashTensor* t : {&x, &y})
      if (const int status = check_cache_tensor(*t, true)) return status;
    if (x.dtype != y.dtype) return SPLASH_ERR_INVALID_ARGUMENT;
    for (int k = 0; k < 4; ++k)
      if (x.size[k] != y.size[k] || (shape != nullptr && k != 1 && x.size[k] != shape->size[k])) return SPLASH_ERR_INVALID_ARGUMENT;
    if (shape != nullptr && x.dtype != shape->dtype) return SPLASH_ERR_INVALID_ARGUMENT;
    if (shape == nullptr) shape = &x;
    if (x.size[1] > 65535) return SPLASH_ERR_TOO_LARGE;
    const int64_t size = x.dtype == SPLASH_F32 ? 4 : 2;
    p.side[i] = {static_cast<const uint8_t*>(x.data), static_cast<uint8_t*>(y.data), x.stride[0] * size, x.stride[1] * size, x.stride[2] * size,
                 y.stride[0] * size, y.stride[1] * size, y.stride[2] * size, (int32_t)x.size[1]};
  }
  if (shape == nullptr) return SPLASH_ERR_INVALID_ARGUMENT;
  if (shape->size[3] % 8 != 0 || a.dim < 2 || a.dim % 2 != 0 || a.dim > shape->size[3]) return SPLASH_ERR_INVALID_ARGUMENT;
  if (shape->size[3] > 256) return SPLASH_ERR_UNSUPPORTED;
  if (a.positions == nullptr || a.turns == nullptr || a.position_stride < 0 || !(a.factor == a.factor)) return SPLASH_ERR_INVALID_ARGUMENT;
  if (shape->size[0] > 0x7fffffffll || shape->size[2] > 0x7fffffffll || shape->size[0] * shape->size[2] > 0x7fffffffll) return SPLASH_ERR_TOO_LARGE;
  p.positions = a.positions;
  p.positions_are_64 = a.positions_are_64;
  p.position_stride = a.position_stride;
  p.turns = a.turns;
  p.rows = (uint32_t)(shape->size[0] * shape->size[2]);
  p.tokens = (uint32_t)shape->size[2];
  p.head_dim = (int32_t)shape->size[3];
  p.dim = a.dim;
  p.factor = a.factor;
  p.sign = a.inverse ? -1.f : 1.f;
  return shape->dtype == SPLASH_BF16  ? pick_rotate<SPLASH_BF16>(p, a.interleaved, stream)
         : shape->dtype == SPLASH_F16 ? pick_rotate<SPLASH_F16>(p, a.interleaved, stream)
                                      : pick_rotate<SPLASH_F32>(p, a.interleaved, stream);
}

}  // namespace sb

extern "C" {

int splash_rotate(const SplashRotateArgs* args, void* cuda_stream) {
  return args == nullptr ? SPLASH_ERR_INVALID_ARGUMENT : sb::rotate(*args, static_cast<cudaStream_t>(cuda_stream));
}

}  // extern "C"
