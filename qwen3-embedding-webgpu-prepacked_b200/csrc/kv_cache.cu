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
// e stops at `low`, where the smallest code times 2^e is the smallest value that is
// left whole: f16's smallest subnormal 2^-24, which attention and conversions keep, but
// bf16's smallest normal 2^-126, so that no value read back depends on how products
// treat f32 subnormals (bf16's range is f32's). Smaller bf16 values are rounded to
// multiples of 2^-126. At the top, where 256 * 2^e (64 * 2^e) would leave the type's
// range, codes stop one step lower (240, 63).
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

  // e of a vector whose largest magnitude is `bits` (of the 16-bit type,
  // finite).
  static __device__ __forceinline__ int exponent(uint32_t bits) {
    const uint32_t u = kBf16 ? bits << 16
                             : __float_as_uint(__half2float(__ushort_as_half(
                                   static_cast<unsigned short>(bits))));
    if (u == 0) return 0;
    if (u < 0x00800000u) return kLow;  // a subnormal bf16
    const int e = static_cast<int>(u >> 23) - 127 - kShift + ((u & 0x7fffffu) > kMantissa ? 1 : 0);
    return e < kLow ? kLow : e;
  }
};

__host__ __device__ constexpr uint32_t kExpBits(bool bf16) { return bf16 ? 0x7f80u : 0x7c00u; }

// Largest magnitude of eight values, as the bits of |x| in both halves: they
// order as the values do, NaN above infinity.
__device__ __forceinline__ uint32_t largest8(const uint4& v) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(v.x & kAbs, v.y & kAbs), __vmaxu2(v.z & kAbs, v.w & kAbs));
}

// The same with NaN left out (one value at a time; NaN is rare).
template <bool kBf16>
__device__ __noinline__ uint32_t largest8_but_nan(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
  for (int i = 0; i < 8; ++i) {
    const uint32_t x = (w[i >> 1] >> (16 * (i & 1))) & 0x7fffu;
    if (x <= kExpBits(kBf16) && x > top) top = x;
  }
  return top | (top << 16);
}

// Codes of eight values by the rule, one value at a time: for vectors with NaN,
// at the top of the range, or too small for the short way below.
template <bool kBf16, int kFormat>
__device__ __noinline__ uint2 encode8_any(uint4 v, int e) {
  using C = Code<kBf16, kFormat>;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const float most = e == C::kTop ? C::kMaxAtTop : C::kMax;
  uint32_t out[2] = {0u, 0u};
  for (int i = 0; i < 8; ++i) {
    const float2 pair = unpack2<kBf16>(w[i >> 1]);
    float x = ((i & 1) ? pair.y : pair.x) * pow2f(-e);
    // comparisons, not fminf: NaN has to stay NaN
    x = x > most ? most : (x < -most ? -most : x);
    uint32_t code;
    if constexpr (kFormat == kKvE4M3) code = float2_to_e4m3x2(x, 0.f) & 0xffu;
    else code = static_cast<uint32_t>(x == x ? __float2int_rn(x) : 0) & 0xffu;
    out[i >> 2] |= code << (8 * (i & 3));
  }
  return make_uint2(out[0], out[1]);
}

// Four codes of two pairs. The products with 2^-e are exact; E4M3 rounds in the
// conversion, INT8 in the sum with 1.5 * 2^m (m: mantissa bits), whose low byte is
// then the code.
template <bool kBf16, int kFormat>
__device__ __forceinline__ uint32_t encode4(uint32_t lo, uint32_t hi, int e) {
  if constexpr (kBf16) {
    const float s = pow2f(-e);
    const float2 a = unpack2<true>(lo), b = unpack2<true>(hi);
    if constexpr (kFormat == kKvE4M3) {
      return float2_to_e4m3x2(a.x * s, a.y * s) | (float2_to_e4m3x2(b.x * s, b.y * s) << 16);
    } else {
      constexpr float kRound = 12582912.f;  // 1.5 * 2^23
      const uint32_t x = __float_as_uint(fmaf(a.x, s, kRound)),
                     y = __float_as_uint(fmaf(a.y, s, kRound)),
                     z = __float_as_uint(fmaf(b.x, s, kRound)),
                     t = __float_as_uint(fmaf(b.y, s, kRound));
      return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, t, 0x0040), 0x5410);
    }
  } else {
    const uint32_t s2 = pair_pow2<false>(-e);
    const __half2 s = *reinterpret_cast<const __half2*>(&s2);
    const __half2 a = *reinterpret_cast<const __half2*>(&lo);
    const __half2 b = *reinterpret_cast<const __half2*>(&hi);
    if constexpr (kFormat == kKvE4M3) {
      const __half2 x = __hmul2(a, s), y = __hmul2(b, s);
      return half2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&x)) |
             (half2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&y)) << 16);
    } else {
      const __half2 round = __floats2half2_rn(1536.f, 1536.f);  // 1.5 * 2^10
      const __half2 x = __hfma2(a, s, round), y = __hfma2(b, s, round);
      return __byte_perm(*reinterpret_cast<const uint32_t*>(&x),
                         *reinterpret_cast<const uint32_t*>(&y), 0x6420);
    }
  }
}

constexpr int kThreads = 128;

// Where vector `vec` of the call is: vectors go head by head through k and then
// v of a token.
struct Where {
  int64_t token;
  int kv, head;
};
__device__ __forceinline__ Where where(const KvCacheArgs& a, uint32_t vec) {
  const uint32_t th = static_cast<uint32_t>((static_cast<uint64_t>(vec) * a.heads_m) >> a.heads_s);
  return {th >> 1, static_cast<int>(th & 1), static_cast<int>(vec - th * a.heads)};
}

// head_dim / 16 lanes hold a vector, 16 values each (two loads, one 16-byte
// store of codes). HBM-bound: a thread's kVectors loads are in flight together, and
// wait for nothing. 80000 tokens of 8 heads into INT8: 81 to 87 us with the clock, 5.7 to 6.1
// TB/s (0.88 to 0.95 of measured; 91 us with divisions by `heads`, which made it bound by
// its arithmetic); 16 tokens: 1.7 us.
template <bool kBf16, int kFormat, int kVectors>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvCacheArgs a) {
  using C = Code<kBf16, kFormat == kKvPlain ? kKvE4M3 : kFormat>;
  const int lanes = a.head_dim / 16, per_pass = kThreads / lanes;
  const int l = threadIdx.x % lanes;
  const uint32_t v0 = blockIdx.x * (per_pass * kVectors) + threadIdx.x / lanes;
  uint4 x[kVectors][2];
  int64_t row[kVectors];  // (slot, head), -1: nothing to write
  bool is_v[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const uint32_t vec = v0 + i * per_pass;
    row[i] = -1;
    is_v[i] = false;
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    if (vec >= a.vectors) continue;
    const Where w = where(a, vec);
    is_v[i] = w.kv;
    // the rows are read whether their slot exists or not: nothing waits for it
    const uint4* src = reinterpret_cast<const uint4*>(
        static_cast<const uint16_t*>(w.kv ? a.v_in : a.k_in) +
        w.token * (w.kv ? a.v_stride : a.k_stride) +
        static_cast<int64_t>(w.head) * a.head_dim + l * 16);
    x[i][0] = __ldcs(src);
    x[i][1] = __ldcs(src + 1);
    const int64_t slot = __ldg(a.slot_of + w.token);
    if (slot >= 0 && slot < a.slots) row[i] = slot * a.heads + w.head;
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const bool v = is_v[i];
    const int64_t at = row[i] * a.head_dim + l * 16;
    if constexpr (kFormat == kKvPlain) {
      if (row[i] >= 0) {
        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(v ? a.v : a.k) + at);
        dst[0] = x[i][0];
        dst[1] = x[i][1];
      }
    } else {
      uint32_t top = __vmaxu2(largest8(x[i][0]), largest8(x[i][1]));
      for (int o = lanes >> 1; o > 0; o >>= 1)
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
      uint32_t bits = max(top & 0xffffu, top >> 16);
      constexpr uint32_t kInf = kExpBits(kBf16);
      const bool nan = bits > kInf;
      if (__any_sync(0xffffffffu, nan)) {
        uint32_t t = __vmaxu2(largest8_but_nan<kBf16>(x[i][0]), largest8_but_nan<kBf16>(x[i][1]));
        for (int o = lanes >> 1; o > 0; o >>= 1)
          t = __vmaxu2(t, __shfl_xor_sync(0xffffffffu, t, o));
        bits = t & 0xffffu;
      }
      if (bits == kInf) bits = kInf - 1;  // infinities count as the largest finite value
      const int e = C::exponent(bits);
      // f16's short way multiplies by 2^-e in f16
      const bool any = nan || e == C::kTop || (!kBf16 && e < -15);
      uint4 code;
      if (any) {
        const uint2 p = encode8_any<kBf16, kFormat>(x[i][0], e);
        const uint2 q = encode8_any<kBf16, kFormat>(x[i][1], e);
        code = make_uint4(p.x, p.y, q.x, q.y);
      } else {
        code.x = encode4<kBf16, kFormat>(x[i][0].x, x[i][0].y, e);
        code.y = encode4<kBf16, kFormat>(x[i][0].z, x[i][0].w, e);
        code.z = encode4<kBf16, kFormat>(x[i][1].x, x[i][1].y, e);
        code.w = encode4<kBf16, kFormat>(x[i][1].z, x[i][1].w, e);
      }
      if (row[i] >= 0) {
        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(v ? a.v : a.k) + at) = code;
        if (l == 0) (v ? a.v_scale : a.k_scale)[row[i]] = static_cast<uint8_t>(e + 127);
      }
    }
  }
}

// The way back: 16 codes a lane (one load, two stores). 8000 scattered slots of 8
// heads from E4M3: 10.8 to 11.2 us, 4.5 TB/s (0.70 of measured; 2 us of it are the launch).
template <bool kBf16, int kFormat, int kVectors>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvCacheArgs a) {
  const int lanes = a.head_dim / 16, per_pass = kThreads / lanes;
  const int l = threadIdx.x % lanes;
  const uint32_t v0 = blockIdx.x * (per_pass * kVectors) + threadIdx.x / lanes;
  uint4 x[kVectors][2];
  int e[kVectors];
  Where at_row[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const uint32_t vec = v0 + i * per_pass;
    x[i][0] = x[i][1] = make_uint4(0u, 0u, 0u, 0u);
    e[i] = 0;
    if (vec >= a.vectors) continue;
    const Where w = at_row[i] = where(a, vec);
    // without a list: the slots from first_slot on, a gap left out after `head`
    const int64_t slot = a.slot_of ? __ldg(a.slot_of + w.token)
                                   : a.first_slot + w.token + (w.token >= a.head ? a.gap : 0);
    if (slot < 0 || slot >= a.slots) continue;  // zeros
    const int64_t row = slot * a.heads + w.head, at = row * a.head_dim + l * 16;
    if constexpr (kFormat == kKvPlain) {
      const uint4* src =
          reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w.kv ? a.v : a.k) + at);
      x[i][0] = src[0];
      x[i][1] = src[1];
    } else {
      x[i][0] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(w.kv ? a.v : a.k) + at);
      e[i] = static_cast<int>((w.kv ? a.v_scale : a.k_scale)[row]) - 127;
    }
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const uint32_t vec = v0 + i * per_pass;
    if (vec >= a.vectors) break;
    const Where w = at_row[i];
    if constexpr (kFormat != kKvPlain) {
      const uint32_t c[4] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w};
      const uint32_t s2 = pair_pow2<kBf16>(e[i]);
      uint32_t y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y[j] = code_pair<kBf16, kFormat == kKvE4M3>((c[j >> 1] >> (16 * (j & 1))) & 0xffffu, s2);
      x[i][0] = make_uint4(y[0], y[1], y[2], y[3]);
      x[i][1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
    const int64_t to = a.slot_of || w.token < a.head ? w.token : w.token + a.gap;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(w.kv ? a.v_out : a.k_out) +
                                          (to * a.heads + w.head) * a.head_dim + l * 16);
    dst[0] = x[i][0];
    dst[1] = x[i][1];
  }
}

template <bool kWrite, bool kBf16, int kVectors>
cudaError_t launch_format(KvCacheArgs a, int format, cudaStream_t stream) {
  kv_cache_divisor(&a);
  const int64_t per_block = kThreads / (a.head_dim / 16) * kVectors;
  const unsigned blocks = static_cast<unsigned>((a.vectors + per_block - 1) / per_block);
  auto go = [&](auto kernel) { kernel<<<blocks, kThreads, 0, stream>>>(a); };
  if constexpr (kWrite) {
    if (format == kKvPlain) go(kv_write_kernel<kBf16, kKvPlain, kVectors>);
    else if (format == kKvE4M3) go(kv_write_kernel<kBf16, kKvE4M3, kVectors>);
    else go(kv_write_kernel<kBf16, kKvInt8, kVectors>);
  } else {
    if (format == kKvPlain) go(kv_read_kernel<kBf16, kKvPlain, kVectors>);
    else if (format == kKvE4M3) go(kv_read_kernel<kBf16, kKvE4M3, kVectors>);
    else go(kv_read_kernel<kBf16, kKvInt8, kVectors>);
  }
  return cudaGetLastError();
}

// Vectors of one lane group. Two where 8-bit rows fill the SMs several times over
// (E4M3 heads of 128, one / two: 16384 tokens of 8 21.2 / 20.0 us, 8192 11.9 / 11.5;
// 4096 7.1 / 7.4, 16 2.0 / 2.7); one for 16-bit rows (16384: 17.7 / 19.9) and in reading,
// whose loads wait for the slot: more groups hide that better (8000: 11.0 / 11.5).
constexpr int64_t kPairLanes = 1 << 20;

}  // namespace

cudaError_t launch_kv_write(const KvCacheArgs& a, int bf16, int format, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  if (format != kKvPlain && static_cast<int64_t>(a.vectors) * (a.head_dim / 16) >= kPairLanes)
    return bf16 ? launch_format<true, true, 2>(a, format, stream)
                : launch_format<true, false, 2>(a, format, stream);
  return bf16 ? launch_format<true, true, 1>(a, format, stream)
              : launch_format<true, false, 1>(a, format, stream);
}
cudaError_t launch_kv_read(const KvCacheArgs& a, int bf16, int format, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  return bf16 ? launch_format<false, true, 1>(a, format, stream)
              : launch_format<false, false, 1>(a, format, stream);
}

}  // namespace qwa
