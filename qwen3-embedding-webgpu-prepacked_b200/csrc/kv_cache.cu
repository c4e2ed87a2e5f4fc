// The key/value cache in 8 bits: quantising rows as they are written, and
// reading them back.
//
// Per (slot, head) vector x[0..d): amax = max |x| (infinities count as the
// type's largest value, NaN not at all), and the scale 2^e is the least power
// of two with amax <= 448 * 2^e (E4M3) or amax <= 127 * 2^e (INT8); 2^0 if
// amax = 0. code = round-to-nearest-even(x * 2^-e). The scale is stored as the
// byte e + 127.
//
// Why powers of two: x * 2^-e is exact, so a value is rounded once and the
// stored codes are the same however they are computed; and code * 2^e is exact
// in f16 and bf16, so an attention that reads the cache works on exactly the
// stored numbers. E4M3 loses nothing by it (a floating format has the same
// relative step under any scale); INT8 loses up to one of its 7 bits.
//
// e stops at `low`, where code * 2^e still is a multiple of the type's
// smallest subnormal, and at the top, where 256 * 2^e (64 * 2^e) would leave
// the type's range, codes stop one step lower (240, 63).
#include <cuda_bf16.h>

#include "convert.cuh"
#include "internal.h"

namespace qwa {
namespace {

template <bool kBf16, int kFormat>
struct Code {
  static constexpr int kTop = (kBf16 ? 127 : 15) - (kFormat == kKvE4M3 ? 7 : 5);
  static constexpr int kLow = kFormat == kKvE4M3 ? (kBf16 ? -117 : -15) : (kBf16 ? -126 : -24);
  static constexpr float kMax = kFormat == kKvE4M3 ? 448.f : 127.f;
  static constexpr float kMaxAtTop = kFormat == kKvE4M3 ? 240.f : 63.f;
  // amax = 1.m * 2^x fits into kMax * 2^e, kMax = 1.75 * 2^8 or 1.984375 * 2^6
  static constexpr int kShift = kFormat == kKvE4M3 ? 8 : 6;
  static constexpr uint32_t kMantissa = kFormat == kKvE4M3 ? 0x600000u : 0x7e0000u;

  // e of a vector whose largest magnitude is amax (an f32 that is a value of
  // the 16-bit type).
  static __device__ __forceinline__ int exponent(float amax) {
    if (amax == 0.f) return 0;
    int x;
    uint32_t m;
    const uint32_t u = __float_as_uint(amax);
    if (u < 0x00800000u) {  // a subnormal bf16
      x = -126;
      m = 0;
    } else {
      x = static_cast<int>(u >> 23) - 127;
      m = u & 0x7fffffu;
    }
    const int e = x - kShift + (m > kMantissa ? 1 : 0);
    return e < kLow ? kLow : e;
  }
};

// Eight values of one lane, and their largest magnitude: infinities count as
// the largest finite value and NaN as nothing.
template <bool kBf16>
__device__ __forceinline__ float largest_of(const uint4& raw, float (&x)[8]) {
  constexpr float kFinite = kBf16 ? 3.3895313892515355e38f : 65504.f;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<kBf16>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
    top = fmaxf(top, fabsf(f.x));  // max(a, NaN) = a
    top = fmaxf(top, fabsf(f.y));
  }
  return fminf(top, kFinite);
}

// Codes of eight values, low byte first.
template <bool kBf16, int kFormat>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], int e) {
  using C = Code<kBf16, kFormat>;
  const float inv_a = pow2f(-(e / 2)), inv_b = pow2f(-(e - e / 2));  // 2^-e may leave f32's range
  const float most = e == C::kTop ? C::kMaxAtTop : C::kMax;
  uint32_t out[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float r[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = x[2 * i + j] * inv_a * inv_b;
      // a comparison, not fminf: NaN has to stay NaN
      r[j] = v > most ? most : (v < -most ? -most : v);
    }
    uint32_t pair;
    if constexpr (kFormat == kKvE4M3) {
      pair = float2_to_e4m3x2(r[0], r[1]);
    } else {
      const int a = r[0] == r[0] ? __float2int_rn(r[0]) : 0;  // NaN: 0
      const int b = r[1] == r[1] ? __float2int_rn(r[1]) : 0;
      pair = (static_cast<uint32_t>(a) & 0xffu) | ((static_cast<uint32_t>(b) & 0xffu) << 8);
    }
    out[i >> 1] |= pair << (16 * (i & 1));
  }
  return make_uint2(out[0], out[1]);
}

template <bool kBf16, int kFormat>
__device__ __forceinline__ uint4 decode8(uint2 codes, int e) {
  const float sa = pow2f(e / 2), sb = pow2f(e - e / 2);
  const uint32_t w[2] = {codes.x, codes.y};
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = w[i >> 1] >> (16 * (i & 1));
    float2 f;
    if constexpr (kFormat == kKvE4M3) {
      f = unpack2<false>(e4m3x2_to_half2(pair));
    } else {
      f = make_float2(static_cast<float>(static_cast<int8_t>(pair & 0xffu)),
                      static_cast<float>(static_cast<int8_t>((pair >> 8) & 0xffu)));
    }
    out[i] = pack2<kBf16>(f.x * sa * sb, f.y * sa * sb);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

constexpr int kThreads = 256;

// d / 8 lanes a vector, one vector of k or v per lane group.
template <bool kBf16, int kFormat>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvCacheArgs a) {
  const int lanes = a.head_dim / 8;
  const int64_t vec = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / lanes;
  const int l = threadIdx.x % lanes;
  const int64_t vectors = static_cast<int64_t>(a.tokens) * a.heads * 2;
  const bool live = vec < vectors;
  const int kv = static_cast<int>(vec & 1);
  const int64_t th = vec >> 1;
  const int64_t t = live ? th / a.heads : 0;
  const int h = live ? static_cast<int>(th % a.heads) : 0;
  const int64_t slot = a.slot_of[t];
  const bool in = live && slot >= 0 && slot < a.slots;
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  const uint16_t* src = static_cast<const uint16_t*>(kv ? a.v_in : a.k_in);
  if (in)
    raw = *reinterpret_cast<const uint4*>(src + t * (kv ? a.v_stride : a.k_stride) +
                                          static_cast<int64_t>(h) * a.head_dim + l * 8);
  const int64_t at = (slot * a.heads + h) * a.head_dim + l * 8;
  if constexpr (kFormat == kKvPlain) {
    if (in) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(kv ? a.v : a.k) + at) = raw;
  } else {
    float x[8];
    float top = largest_of<kBf16>(raw, x);
    for (int o = lanes >> 1; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = Code<kBf16, kFormat>::exponent(top);
    if (in) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(kv ? a.v : a.k) + at) =
          encode8<kBf16, kFormat>(x, e);
      if (l == 0) (kv ? a.v_scale : a.k_scale)[slot * a.heads + h] = static_cast<uint8_t>(e + 127);
    }
  }
}

template <bool kBf16, int kFormat>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvCacheArgs a) {
  const int lanes = a.head_dim / 8;
  const int64_t vec = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / lanes;
  const int l = threadIdx.x % lanes;
  if (vec >= static_cast<int64_t>(a.tokens) * a.heads * 2) return;
  const int kv = static_cast<int>(vec & 1);
  const int64_t t = (vec >> 1) / a.heads;
  const int h = static_cast<int>((vec >> 1) % a.heads);
  const int64_t slot = a.slot_of[t];
  uint4 out = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0 && slot < a.slots) {
    const int64_t at = (slot * a.heads + h) * a.head_dim + l * 8;
    if constexpr (kFormat == kKvPlain) {
      out = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(kv ? a.v : a.k) + at);
    } else {
      const uint2 codes =
          *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(kv ? a.v : a.k) + at);
      const int e = static_cast<int>((kv ? a.v_scale : a.k_scale)[slot * a.heads + h]) - 127;
      out = decode8<kBf16, kFormat>(codes, e);
    }
  }
  uint16_t* dst = static_cast<uint16_t*>(kv ? a.v_out : a.k_out);
  *reinterpret_cast<uint4*>(dst + (t * a.heads + h) * a.head_dim + l * 8) = out;
}

template <bool kWrite, bool kBf16>
cudaError_t launch_format(const KvCacheArgs& a, int format, cudaStream_t stream) {
  const int64_t threads = static_cast<int64_t>(a.tokens) * a.heads * 2 * (a.head_dim / 8);
  const unsigned blocks = static_cast<unsigned>((threads + kThreads - 1) / kThreads);
  auto go = [&](auto kernel) { kernel<<<blocks, kThreads, 0, stream>>>(a); };
  if constexpr (kWrite) {
    if (format == kKvPlain) go(kv_write_kernel<kBf16, kKvPlain>);
    else if (format == kKvE4M3) go(kv_write_kernel<kBf16, kKvE4M3>);
    else go(kv_write_kernel<kBf16, kKvInt8>);
  } else {
    if (format == kKvPlain) go(kv_read_kernel<kBf16, kKvPlain>);
    else if (format == kKvE4M3) go(kv_read_kernel<kBf16, kKvE4M3>);
    else go(kv_read_kernel<kBf16, kKvInt8>);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_write(const KvCacheArgs& a, int bf16, int format, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  return bf16 ? launch_format<true, true>(a, format, stream)
              : launch_format<true, false>(a, format, stream);
}
cudaError_t launch_kv_read(const KvCacheArgs& a, int bf16, int format, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  return bf16 ? launch_format<false, true>(a, format, stream)
              : launch_format<false, false>(a, format, stream);
}

}  // namespace qwa
