// Rotary positions: the (cos, sin) table and its application to q and k.
//
// Table: table[p][i] = (m cos(a), m sin(a)), a = (first + p) * f_i in 64 bits,
// rounded once to f32. It generalises src/webgpu/model.ts:76-83, whose table
// has f_i = theta^(-i/64) and m = 1; scaled contexts give other f_i and m
// (rope_frequencies in api.cu).
//
// Rotation of the first `rotary` values of a head, pairs (x1, x2) =
// (x[i], x[i + rotary/2]) or (x[2i], x[2i+1]):
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s      (inverse: s -> -s)
// in f32, rounded once. The rotation is orthogonal up to the factor m, so the
// inverse is also the operator's gradient (dx from dy).
#include <cuda_bf16.h>

#include "convert.cuh"
#include "internal.h"

namespace qwa {
namespace {

// ------------------------------------------------------------------- table
// A thread takes one frequency over kTableRun positions: sin and cos of the
// first, then turns by f in 64 bits (16 turns add less than 2^-47, far below the
// rounding to f32). With sincos for every entry the kernel was bound by its 64-bit
// arithmetic (27 us for 131072 x 64 entries); now by its writes (12.4 us, 5.4 TB/s, 0.84
// of measured; runs of 8, 32 and 64 positions took 13.6, 12.9 and 12.8).
constexpr int kTableRun = 16;
constexpr int kTableThreads = 128;

__global__ void __launch_bounds__(kTableThreads)
    rope_table_kernel(const __grid_constant__ RopeFrequencies fr, float2* __restrict__ table,
                      int64_t first, int positions) {
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kTableThreads + threadIdx.x;
  const int i = static_cast<int>(idx % fr.half);
  const int64_t p0 = idx / fr.half * kTableRun;
  if (p0 >= positions) return;
  const double f = fr.f[i];
  const int n = static_cast<int>(positions - p0 < kTableRun ? positions - p0 : kTableRun);
  float2* dst = table + p0 * fr.half + i;
  double s, c, sf, cf;
  sincos(static_cast<double>(first + p0) * f, &s, &c);
  sincos(f, &sf, &cf);
  s *= fr.m;
  c *= fr.m;
  for (int j = 0; j < n; ++j) {
    *dst = make_float2(static_cast<float>(c), static_cast<float>(s));
    dst += fr.half;
    const double next = c * cf - s * sf;
    s = s * cf + c * sf;
    c = next;
  }
}

// ---------------------------------------------------------------- rotation
constexpr int kRopeThreads = 256;
// shared memory of a token's cosines and sines, whole 16-byte units
__host__ __device__ constexpr int rope_table_bytes(int half) { return (half * 8 + 15) / 16 * 16; }

// One block a token: what turns passes through shared memory, so pairs of any
// distance and rows of any stride and alignment are served. kUnits: rows of whole 16-byte
// units, moved as such; the units behind the rotated part go straight through.
// 8000 tokens of 16 + 8 heads of 128, 34 in halves: 31 us, 3.2 TB/s; rows of an odd stride, value
// by value: 113 us, 0.87 TB/s (all 128 in halves 118). Bound by its passes through shared memory,
// value by value by 2-byte accesses.
template <typename T, bool kUnits>
__global__ void __launch_bounds__(kRopeThreads) rope_any_kernel(const RopeArgs a) {
  extern __shared__ __align__(16) uint8_t rope_smem[];
  const int t = blockIdx.x;
  const int pos = a.positions[t];
  if (pos < 0 || pos >= a.table_rows) return;
  const int half = a.rotary / 2, d = a.head_dim;
  const bool inter = a.layout == 1;
  float2* cs = reinterpret_cast<float2*>(rope_smem);  // [half], then the values
  T* x = reinterpret_cast<T*>(rope_smem + rope_table_bytes(half));
  const float2* row = a.table + static_cast<int64_t>(pos) * half;
  for (int i = threadIdx.x; i < half; i += kRopeThreads) {
    const float2 v = __ldg(row + i);
    cs[i] = make_float2(v.x, a.inverse ? -v.y : v.y);
  }
  // value c < rotary of the head whose values begin at h
  auto turned = [&](const T* h, int c) -> T {
    const int i = inter ? c >> 1 : (c < half ? c : c - half);
    const bool first = inter ? (c & 1) == 0 : c < half;
    const int far = inter ? 1 : half;
    const float2 v = cs[i];
    const float mine = to_float(h[c]), other = to_float(h[first ? c + far : c - far]);
    return from_float<T>(first ? mine * v.x - other * v.y : mine * v.x + other * v.y);
  };
  const int heads = a.q.heads + a.k.heads;
  // heads are taken as many at a time as fit the block's shared memory
  for (int h0 = 0; h0 < heads; h0 += a.smem_heads) {
    const int nh = min(a.smem_heads, heads - h0);
    __syncthreads();
    if constexpr (kUnits) {
      const int units = d / 8, turning = (a.rotary + 7) / 8;  // of a head
      uint4* xs = reinterpret_cast<uint4*>(x);
      for (int e = threadIdx.x; e < nh * units; e += kRopeThreads) {
        const int h = e / units, u = e - h * units;
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(a.in_row(t, h0 + h)) + u);
        if (u < turning) xs[h * turning + u] = v;
        else reinterpret_cast<uint4*>(a.out_row(t, h0 + h))[u] = v;
      }
      __syncthreads();
      for (int e = threadIdx.x; e < nh * turning; e += kRopeThreads) {
        const int h = e / turning, u = e - h * turning;
        const T* head = x + h * turning * 8;
        uint4 v = xs[e];
        T y[8];
        memcpy(y, &v, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (u * 8 + j < a.rotary) y[j] = turned(head, u * 8 + j);
        memcpy(&v, y, 16);
        reinterpret_cast<uint4*>(a.out_row(t, h0 + h))[u] = v;
      }
    } else {
      for (int e = threadIdx.x; e < nh * d; e += kRopeThreads)
        x[e] = reinterpret_cast<const T*>(a.in_row(t, h0 + e / d))[e % d];
      __syncthreads();
      for (int e = threadIdx.x; e < nh * d; e += kRopeThreads) {
        const int h = e / d, c = e - h * d;
        reinterpret_cast<T*>(a.out_row(t, h0 + h))[c] = c < a.rotary ? turned(x + h * d, c) : x[e];
      }
    }
  }
}

// Rows of whole 16-byte units. A thread owns one unit u of the heads hs, hs +
// step, ... of a token, so its cosines and sines are read once. Units of a head:
//   half:        u < rotary / 16: the 8 pairs from 8 u on (two 16-byte loads);
//                then the units behind the rotated part, copied
//   interleaved: 4 pairs, of which those past the rotated part are copied
// HBM-bound: a thread issues the loads of kHeads heads before any arithmetic,
// six in both layouts (two to eight, and blocks of 96 to 256, were slower). Loading
// before the position is known cost registers and was slower too (25 us against 20).
// 8000 tokens of 16 + 8 heads, f16 in halves: 19.8 us, 5.2 TB/s (0.80 of measured);
// 20011 in bf16, half of each head: 44.3 us, 5.7 TB/s (0.88); 16 tokens: 2.2 us.
constexpr int kRowThreads = 128;

template <bool kBf16>
__device__ __forceinline__ uint32_t turn_pair(uint32_t x, float c, float s) {
  const float2 v = unpack2<kBf16>(x);
  return pack2<kBf16>(v.x * c - v.y * s, v.y * c + v.x * s);
}

template <bool kBf16, bool kInterleaved>
__global__ void __launch_bounds__(kRowThreads) rope_rows_kernel(const RopeArgs a) {
  constexpr int kHeads = kInterleaved ? 6 : 3;
  const int group = threadIdx.x / a.token_threads;  // token of the block
  const int r = threadIdx.x - group * a.token_threads;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * a.block_tokens + group;
  if (group >= a.block_tokens || t >= a.tokens) return;
  const int u = r % a.units, hs = r / a.units;
  const int pos = __ldg(a.positions + t);
  if (pos < 0 || pos >= a.table_rows) return;
  const int half = a.rotary / 2, heads = a.q.heads + a.k.heads;
  const float2* row = a.table + static_cast<int64_t>(pos) * half;
  const bool turns = kInterleaved ? u * 4 < half : u * 8 < half;
  // first value of the unit
  const int at = kInterleaved || turns ? u * 8 : a.rotary + (u - half / 8) * 8;
  constexpr int kPairs = kInterleaved ? 4 : 8;
  float c[kPairs], s[kPairs];
  if (turns) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const bool in = !kInterleaved || u * 4 + i < half;
      const float2 cs = in ? __ldg(row + u * kPairs + i) : make_float2(1.f, 0.f);
      c[i] = cs.x;
      s[i] = a.inverse ? -cs.y : cs.y;
    }
  }
  for (int h0 = hs; h0 < heads; h0 += kHeads * a.head_step) {
    uint4 x[kHeads], y[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i * a.head_step;
      if (h < heads) {
        const uint16_t* src = a.in_row(t, h) + at;
        x[i] = __ldcs(reinterpret_cast<const uint4*>(src));
        if (!kInterleaved && turns) y[i] = __ldcs(reinterpret_cast<const uint4*>(src + half));
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i * a.head_step;
      if (h >= heads) break;
      uint16_t* dst = a.out_row(t, h) + at;
      if (turns) {
        uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        if constexpr (kInterleaved) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t turned = turn_pair<kBf16>(xs[j], c[j], s[j]);
            if (u * 4 + j < half) xs[j] = turned;
          }
        } else {
          uint32_t ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 p = unpack2<kBf16>(xs[j]), q = unpack2<kBf16>(ys[j]);
            const float c0 = c[2 * j], c1 = c[2 * j + 1], s0 = s[2 * j], s1 = s[2 * j + 1];
            xs[j] = pack2<kBf16>(p.x * c0 - q.x * s0, p.y * c1 - q.y * s1);
            ys[j] = pack2<kBf16>(q.x * c0 + p.x * s0, q.y * c1 + p.y * s1);
          }
          *reinterpret_cast<uint4*>(dst + half) = make_uint4(ys[0], ys[1], ys[2], ys[3]);
        }
        x[i] = make_uint4(xs[0], xs[1], xs[2], xs[3]);
      }
      *reinterpret_cast<uint4*>(dst) = x[i];
    }
  }
}

bool whole_units(const RopeSide& s) {
  auto multiple = [](const void* p, int64_t a, int64_t b) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && a % 8 == 0 && b % 8 == 0;
  };
  return s.heads == 0 || (multiple(s.in, s.in_stride, s.in_head_stride) &&
                          multiple(s.out, s.out_stride, s.out_head_stride));
}

}  // namespace

cudaError_t launch_rope_table(const RopeFrequencies& fr, float2* table, int64_t first,
                              int positions, cudaStream_t stream) {
  if (positions <= 0) return cudaSuccess;
  const int64_t runs = (static_cast<int64_t>(positions) + kTableRun - 1) / kTableRun;
  const int64_t blocks = (runs * fr.half + kTableThreads - 1) / kTableThreads;
  rope_table_kernel<<<static_cast<unsigned>(blocks), kTableThreads, 0, stream>>>(fr, table, first,
                                                                                positions);
  return cudaGetLastError();
}

cudaError_t launch_rope(RopeArgs a, int bf16, cudaStream_t stream) {
  const int heads = a.q.heads + a.k.heads;
  if (a.tokens <= 0 || heads <= 0) return cudaSuccess;
  const bool whole = a.head_dim % 8 == 0 && whole_units(a.q) && whole_units(a.k);
  // without shared memory, pairs of halves need whole units on both sides; pairs
  // of neighbours never straddle one
  const bool rows = whole && a.head_dim <= 8 * kRowThreads &&
                    (a.layout == 1 || a.rotary % 16 == 0);
  if (rows) {
    a.units = a.layout == 1 ? a.head_dim / 8 : a.rotary / 16 + (a.head_dim - a.rotary) / 8;
    // Heads of one thread: one until such threads fill the SMs (16 + 8 heads of 128
    // in halves: 64 tokens 2.3 us against 2.5, 512 3.8 / 3.9, 1024 4.9 / 4.9), then as
    // many as it has loads in flight for, so that fewer threads read a token's
    // cosines (2048: 7.6 against 6.8, 4096: 12.6 / 10.8).
    const int most = a.layout == 1 ? 6 : 3;
    const bool few = static_cast<int64_t>(a.tokens) * heads * a.units < 200000;
    const int step = few ? heads : (heads + most - 1) / most;
    a.head_step = step * a.units <= kRowThreads ? step : kRowThreads / a.units;
    a.token_threads = a.units * a.head_step;
    a.block_tokens = kRowThreads / a.token_threads;
    const unsigned blocks = static_cast<unsigned>((a.tokens + a.block_tokens - 1) / a.block_tokens);
    auto go = [&](auto kernel) { kernel<<<blocks, kRowThreads, 0, stream>>>(a); };
    if (bf16) a.layout == 1 ? go(rope_rows_kernel<true, true>) : go(rope_rows_kernel<true, false>);
    else a.layout == 1 ? go(rope_rows_kernel<false, true>) : go(rope_rows_kernel<false, false>);
    return cudaGetLastError();
  }
  a.smem_heads = 32768 / (a.head_dim * 2);
  if (a.smem_heads > heads) a.smem_heads = heads;
  const size_t smem = rope_table_bytes(a.rotary / 2) +
                      static_cast<size_t>(a.smem_heads) * a.head_dim * 2;
  auto go = [&](auto kernel) { kernel<<<a.tokens, kRopeThreads, smem, stream>>>(a); };
  if (bf16) whole ? go(rope_any_kernel<__nv_bfloat16, true>) : go(rope_any_kernel<__nv_bfloat16, false>);
  else whole ? go(rope_any_kernel<__half, true>) : go(rope_any_kernel<__half, false>);
  return cudaGetLastError();
}

}  // namespace qwa
