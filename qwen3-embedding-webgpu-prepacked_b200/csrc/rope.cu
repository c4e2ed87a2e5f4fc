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
constexpr int kTableRun = 16;       // consecutive positions of one thread
constexpr int kTableThreads = 256;

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
  for (int j = 0; j < n; ++j) {
    double s, c;
    sincos(static_cast<double>(first + p0 + j) * f, &s, &c);
    dst[static_cast<int64_t>(j) * fr.half] =
        make_float2(static_cast<float>(c * fr.m), static_cast<float>(s * fr.m));
  }
}

// ---------------------------------------------------------------- rotation
constexpr int kRopeThreads = 256;

// One block a token; the token's heads pass through shared memory, so pairs of
// any distance and any stride or alignment are served.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_any_kernel(const RopeArgs a) {
  extern __shared__ __align__(16) uint8_t rope_smem[];
  T* x = reinterpret_cast<T*>(rope_smem);
  const int t = blockIdx.x;
  const int pos = a.positions[t];
  if (pos < 0 || pos >= a.table_rows) return;
  const int half = a.rotary / 2, d = a.head_dim;
  const float2* row = a.table + static_cast<int64_t>(pos) * half;
  // heads are taken as many at a time as fit the block's shared memory
  for (int h0 = 0; h0 < a.q.heads + a.k.heads; h0 += a.smem_heads) {
    const int nh = min(a.smem_heads, a.q.heads + a.k.heads - h0);
    __syncthreads();
    for (int e = threadIdx.x; e < nh * d; e += kRopeThreads) {
      const int h = h0 + e / d;
      x[e] = reinterpret_cast<const T*>(a.in_row(t, h))[e % d];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nh * d; e += kRopeThreads) {
      const int h = h0 + e / d, c = e % d;
      T* out = reinterpret_cast<T*>(a.out_row(t, h));
      if (c >= a.rotary) {
        out[c] = x[e];
        continue;
      }
      const bool inter = a.layout == 1;
      const int i = inter ? c >> 1 : (c < half ? c : c - half);
      const bool first = inter ? (c & 1) == 0 : c < half;
      const float2 cs = __ldg(row + i);
      const float sn = a.inverse ? -cs.y : cs.y;
      const float mine = to_float(x[e]);
      const float other = to_float(x[first ? e + (inter ? 1 : half) : e - (inter ? 1 : half)]);
      out[c] = from_float<T>(first ? mine * cs.x - other * sn : mine * cs.x + other * sn);
    }
  }
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
  if (a.tokens <= 0 || a.q.heads + a.k.heads <= 0) return cudaSuccess;
  a.smem_heads = 32768 / (a.head_dim * 2);
  const int heads = a.q.heads + a.k.heads;
  if (a.smem_heads > heads) a.smem_heads = heads;
  const size_t smem = static_cast<size_t>(a.smem_heads) * a.head_dim * 2;
  if (bf16)
    rope_any_kernel<__nv_bfloat16><<<a.tokens, kRopeThreads, smem, stream>>>(a);
  else
    rope_any_kernel<__half><<<a.tokens, kRopeThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace qwa
