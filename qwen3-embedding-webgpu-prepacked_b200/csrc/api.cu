// Host side of the C ABI declared in include/qwa.h.
//
// A context (qwa_ctx) owns, per device: the RoPE cos/sin table
// (src/webgpu/model.ts:76-83, rebuilt when a longer sequence arrives), a
// device status word that kernels write on a failed bounded wait, and a cache
// of launch plans keyed by (cu_seqlens, resolved mode, prefix, window) -- the
// counterpart of the reference engine's plan cache per "batch:sequence"
// (src/webgpu/embedding-engine.ts:70-75). A plan holds the device copy of
// cu_seqlens and the attention work list sorted longest-first.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <exception>
#include <functional>
#include <map>
#include <memory>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/qwa.h"
#include "internal.h"
#include "prefix_attention.h"
#include "ptx.cuh"

using namespace qwa;

namespace {

constexpr size_t kMaxPlans = 64;

struct Plan {
  int32_t* d_cu = nullptr;
  AttnItem* d_items = nullptr;   // grouped by CTA, then the CTAs' first items (int)
  const int* d_offsets = nullptr;  // inside d_items: CTA c runs items [off[c], off[c+1])
  int n_items = 0;
  int n_ctas = 0;
  int batch = 0;
  int total = 0;
  int max_len = 0;
  ~Plan() {
    if (d_cu) cudaFree(d_cu);
    if (d_items) cudaFree(d_items);
  }
};

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

}  // namespace

struct qwa_ctx {
  int device = 0;
  int sms = 148;  // persistent attention grid size
  std::string error;
  int* d_status = nullptr;
  float* d_rope = nullptr;
  int rope_positions = 0;
  float rope_theta = 0.f;
  std::map<std::vector<int32_t>, std::unique_ptr<Plan>> plans;
  std::vector<std::vector<int32_t>> plan_order;  // insertion order for eviction
  // f16 weights dequantised from Q4_0 tile32 buffers, keyed by (buffer, n, k)
  std::map<std::tuple<const void*, int, int>, __half*> weights;
  std::vector<__half*> retired;  // forgotten copies, freed outside stream capture
  unsigned long long* trace = nullptr;           // QWA_TRACE builds only
  unsigned long long wait_ns = kWaitTimeoutNs;    // bounded-wait limit of the attention kernel
  int skip_load = -1;                             // test hook, see qwa_set_debug
  float* small_ws = nullptr;                      // partial sums of the small-M Q4_0 path
  size_t small_ws_bytes = 0;
  int clusters[9] = {};           // [n]: clusters of n CTAs that run at one time
  cudaStream_t upload = nullptr;  // copies of prefix plans, waited for before they are used
};

// Work lists of a shared-prefix attention, owned by the caller.
struct qwa_prefix_plan {
  int device = 0;
  PrefixShape shape{};
  int total_q = 0, total_k = 0;
  void* memory = nullptr;  // items, tiles, rows, offsets
  const PrefixItem* items = nullptr;
  const PrefixTile* tiles = nullptr;
  const PrefixRow* rows = nullptr;
  const int* offsets = nullptr;
  int grid = 0, splits = 1;
  int blocks = 0;                // blocks of rows, each with all kv heads
  int gap_beg = 0, gap_end = 0;  // prefix keys that no tile reaches
};

namespace {

qwa_status fail(qwa_ctx* ctx, qwa_status st, const char* fmt, ...) __attribute__((format(printf, 3, 4)));
qwa_status fail(qwa_ctx* ctx, qwa_status st, const char* fmt, ...) {
  if (ctx) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    ctx->error = buf;
  }
  return st;
}

#define QWA_CUDA(ctx, call)                                                                 \
  do {                                                                                      \
    cudaError_t e_ = (call);                                                                \
    if (e_ != cudaSuccess)                                                                  \
      return fail(ctx, QWA_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));       \
  } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

qwa_status ensure_encode(qwa_ctx* ctx) {
  if (g_encode) return QWA_OK;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
  if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn)
    return fail(ctx, QWA_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  return QWA_OK;
}

// 3-D 16-bit map {128 dims, heads, rows}: head stride 256 B, row stride
// row_stride_bytes; box {64, box_heads, box_rows} with 128-byte swizzle, so one
// load lands as box_rows * box_heads rows x 128 B (the canonical SW128 K-major
// atom layout), heads innermost.
qwa_status make_map(qwa_ctx* ctx, CUtensorMap* map, const void* base, int heads, int64_t rows,
                    int64_t row_stride_bytes, uint32_t box_rows = 128, uint32_t box_heads = 1,
                    bool bf16 = false) {
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {256, static_cast<cuuint64_t>(row_stride_bytes)};
  cuuint32_t box[3] = {64, box_heads, box_rows};
  cuuint32_t elem[3] = {1, 1, 1};
  const CUtensorMapDataType type =
      bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = g_encode(map, type, 3, const_cast<void*>(base), dims,
                        strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(ctx, QWA_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return QWA_OK;
}

// 2-D f16 map {inner, rows} with row stride inner*2 bytes, box {64, box_rows},
// 128-byte swizzle (one box = box_rows rows x 128 B, the SW128 K-major atom
// layout the GEMM's descriptors expect). Rows past `rows` read as zero.
qwa_status make_map_2d(qwa_ctx* ctx, CUtensorMap* map, const void* base, int64_t inner,
                       int64_t rows, uint32_t box_rows) {
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(inner * 2)};
  cuuint32_t box[2] = {64, box_rows};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims,
                        strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(ctx, QWA_ERR_CUDA, "cuTensorMapEncodeTiled (2-D) failed (%d)", static_cast<int>(r));
  return QWA_OK;
}

// Output maps of the fused QKV epilogue: boxes of 32 elements x 32 rows
// (64-byte rows, 64-byte swizzle). heads == 0: 2-D {inner, rows}; otherwise
// 3-D {128, heads, rows} with a 256-byte head stride.
qwa_status make_out_map(qwa_ctx* ctx, CUtensorMap* map, void* base, int64_t inner, int heads,
                        int64_t rows, int64_t row_stride_bytes) {
  CUresult r;
  if (heads == 0) {
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_stride_bytes)};
    cuuint32_t box[2] = {32, 32};
    cuuint32_t elem[2] = {1, 1};
    r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, dims, strides, box, elem,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[2] = {256, static_cast<cuuint64_t>(row_stride_bytes)};
    cuuint32_t box[3] = {32, 1, 32};
    cuuint32_t elem[3] = {1, 1, 1};
    r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, elem,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  if (r != CUDA_SUCCESS)
    return fail(ctx, QWA_ERR_CUDA, "cuTensorMapEncodeTiled (output) failed (%d)",
                static_cast<int>(r));
  return QWA_OK;
}

qwa_status check_cu(qwa_ctx* ctx, const int32_t* cu, int batch, int* total, int* max_len) {
  if (!cu) return fail(ctx, QWA_ERR_INVALID_ARG, "cu_seqlens_host is NULL");
  if (batch < 1) return fail(ctx, QWA_ERR_INVALID_ARG, "batch must be >= 1 (got %d)", batch);
  if (cu[0] != 0) return fail(ctx, QWA_ERR_INVALID_ARG, "cu_seqlens[0] must be 0");
  int ml = 0;
  for (int b = 0; b < batch; ++b) {
    if (cu[b + 1] < cu[b])
      return fail(ctx, QWA_ERR_INVALID_ARG, "cu_seqlens must be non-decreasing (index %d)", b + 1);
    ml = std::max(ml, cu[b + 1] - cu[b]);
  }
  *total = cu[batch];
  *max_len = ml;
  return QWA_OK;
}

// Work schedule of an attention call. Items are one 128-row query tile x one
// kv head; each gets a cost in key-tile periods (narrow tiles cost less, every
// item pays a fixed fill/drain share). The items are dealt to `sms` CTAs by
// list scheduling (each to the least-loaded CTA) in this order:
// * longest first, which bounds the final imbalance (LPT);
// * for full-causal calls on long requests, request batches first: the items
//   of a few requests whose K/V fit well inside L2 are dealt before the next
//   batch's, so the CTAs running at one time read the same K/V (longest first
//   within a batch). Without it every wave touches every request's K/V and
//   the K/V of earlier keys is re-read from HBM once per query tile.
// Returns the items grouped by CTA and offsets[c]..offsets[c+1] per CTA.
constexpr double kItemOverhead = 0.6;                   // periods per item
constexpr int kGroupMinLen = 2048;                      // full causal, longest request
constexpr int64_t kGroupKvBytes = 48ll << 20;           // K/V bytes per request batch
std::vector<AttnItem> schedule_work(const int32_t* cu, int batch, int sparse, int prefix,
                                    int window, int sms, std::vector<int>* offsets) {
  struct Work {
    double cost;
    int group;
    AttnItem item;
  };
  int max_len = 0;
  for (int b = 0; b < batch; ++b) max_len = std::max(max_len, cu[b + 1] - cu[b]);
  const bool grouped = !sparse && max_len >= kGroupMinLen;
  std::vector<Work> work;
  int group = 0;
  int64_t group_bytes = 0;
  for (int b = 0; b < batch; ++b) {
    const int len = cu[b + 1] - cu[b];
    const int64_t kv_bytes = static_cast<int64_t>(len) * kKVHeads * kHeadDim * 2 * 2;
    if (grouped && group_bytes > 0 && group_bytes + kv_bytes > kGroupKvBytes) {
      ++group;
      group_bytes = 0;
    }
    group_bytes += kv_bytes;
    for (int q0 = 0; q0 < len; q0 += kBlockM) {
      const KeySchedule s = make_key_schedule(q0, len, sparse, prefix, window);
      const int q_last = std::min(q0 + kBlockM, len) - 1;
      double cost = kItemOverhead;
      for (int j = 0; j < s.n; ++j)
        cost += 0.35 + 0.65 * key_tile_width(s, j, q_last, prefix) / double(kBlockN);
      for (int g = 0; g < kKVHeads; ++g)
        work.push_back({cost, grouped ? group : 0, make_int4(cu[b] + q0, q0, len, g)});
    }
  }
  std::stable_sort(work.begin(), work.end(), [](const Work& a, const Work& b) {
    return a.group != b.group ? a.group < b.group : a.cost > b.cost;
  });
  const int n_ctas = static_cast<int>(std::min<size_t>(work.size(), static_cast<size_t>(sms)));
  std::vector<std::vector<int>> per_cta(n_ctas);
  // min-heap of (load, cta)
  std::vector<std::pair<double, int>> heap;
  for (int c = 0; c < n_ctas; ++c) heap.push_back({0.0, c});
  auto cmp = [](const std::pair<double, int>& a, const std::pair<double, int>& b) {
    return a.first != b.first ? a.first > b.first : a.second > b.second;
  };
  std::make_heap(heap.begin(), heap.end(), cmp);
  for (size_t i = 0; i < work.size(); ++i) {
    std::pop_heap(heap.begin(), heap.end(), cmp);
    auto& top = heap.back();
    per_cta[top.second].push_back(static_cast<int>(i));
    top.first += work[i].cost;
    std::push_heap(heap.begin(), heap.end(), cmp);
  }
  std::vector<AttnItem> items;
  items.reserve(work.size());
  offsets->assign(1, 0);
  for (int c = 0; c < n_ctas; ++c) {
    for (int i : per_cta[c]) items.push_back(work[i].item);
    offsets->push_back(static_cast<int>(items.size()));
  }
  return items;
}

// Plan lookup/creation. sparse < 0 requests a plan without attention items
// (the prologue only needs the device cu_seqlens).
qwa_status get_plan(qwa_ctx* ctx, const int32_t* cu, int batch, int sparse, int prefix,
                    int window, cudaStream_t stream, Plan** out) {
  std::vector<int32_t> key;
  key.reserve(batch + 4);
  key.push_back(sparse);
  key.push_back(prefix);
  key.push_back(window);
  key.insert(key.end(), cu, cu + batch + 1);
  auto it = ctx->plans.find(key);
  if (it != ctx->plans.end()) {
    *out = it->second.get();
    return QWA_OK;
  }
  auto plan = std::make_unique<Plan>();
  plan->batch = batch;
  plan->total = cu[batch];
  for (int b = 0; b < batch; ++b) plan->max_len = std::max(plan->max_len, cu[b + 1] - cu[b]);
  QWA_CUDA(ctx, cudaMalloc(&plan->d_cu, sizeof(int32_t) * (batch + 1)));
  QWA_CUDA(ctx, cudaMemcpyAsync(plan->d_cu, cu, sizeof(int32_t) * (batch + 1),
                                cudaMemcpyHostToDevice, stream));
  if (sparse >= 0) {
    std::vector<int> offsets;
    std::vector<AttnItem> items = schedule_work(cu, batch, sparse, prefix, window, ctx->sms,
                                                &offsets);
    plan->n_items = static_cast<int>(items.size());
    plan->n_ctas = static_cast<int>(offsets.size()) - 1;
    if (!items.empty()) {
      const size_t item_bytes = sizeof(AttnItem) * items.size();
      const size_t bytes = item_bytes + sizeof(int) * offsets.size();
      std::vector<uint8_t> host(bytes);
      std::memcpy(host.data(), items.data(), item_bytes);
      std::memcpy(host.data() + item_bytes, offsets.data(), sizeof(int) * offsets.size());
      QWA_CUDA(ctx, cudaMalloc(&plan->d_items, bytes));
      QWA_CUDA(ctx, cudaMemcpyAsync(plan->d_items, host.data(), bytes, cudaMemcpyHostToDevice,
                                    stream));
      // pageable source: the copy is staged before cudaMemcpyAsync returns
      plan->d_offsets = reinterpret_cast<const int*>(
          reinterpret_cast<const uint8_t*>(plan->d_items) + item_bytes);
    }
  }
  if (ctx->plans.size() >= kMaxPlans) {
    // Evict the oldest plan; cudaFree synchronises, so no launch still uses it.
    ctx->plans.erase(ctx->plan_order.front());
    ctx->plan_order.erase(ctx->plan_order.begin());
  }
  *out = plan.get();
  ctx->plan_order.push_back(key);
  ctx->plans.emplace(std::move(key), std::move(plan));
  return QWA_OK;
}

// RoPE table of src/webgpu/model.ts:76-83: angle = pos * theta^(-d/64) in
// double, stored as f32 (cos, sin) pairs.
qwa_status ensure_rope(qwa_ctx* ctx, int positions, float theta, cudaStream_t stream) {
  if (positions <= ctx->rope_positions && theta == ctx->rope_theta) return QWA_OK;
  int n = std::max(positions, 1);
  if (theta == ctx->rope_theta) n = std::max(n, 2 * ctx->rope_positions);
  std::vector<float> host(static_cast<size_t>(n) * 128);
  for (int p = 0; p < n; ++p)
    for (int d = 0; d < 64; ++d) {
      const double angle = static_cast<double>(p) * std::pow(static_cast<double>(theta), -d / 64.0);
      host[(static_cast<size_t>(p) * 64 + d) * 2] = static_cast<float>(std::cos(angle));
      host[(static_cast<size_t>(p) * 64 + d) * 2 + 1] = static_cast<float>(std::sin(angle));
    }
  if (ctx->d_rope) {
    cudaFree(ctx->d_rope);
    ctx->d_rope = nullptr;
    ctx->rope_positions = 0;
  }
  QWA_CUDA(ctx, cudaMalloc(&ctx->d_rope, host.size() * sizeof(float)));
  QWA_CUDA(ctx, cudaMemcpyAsync(ctx->d_rope, host.data(), host.size() * sizeof(float),
                                cudaMemcpyHostToDevice, stream));
  // The pageable copy above has been staged before return; keep ordering simple.
  QWA_CUDA(ctx, cudaStreamSynchronize(stream));
  ctx->rope_positions = n;
  ctx->rope_theta = theta;
  return QWA_OK;
}

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    cudaGetDevice(&cur);
    if (prev >= 0 && cur != prev) cudaSetDevice(prev);
  }
};

qwa_status run_prologue(qwa_ctx* ctx, const void* qkv, int64_t qkv_stride, const float* q_weight,
                        const float* k_weight, void* q_out, void* k_out, const int32_t* d_cu,
                        int batch, int tokens, int padded_sequence, int positions, float eps,
                        float theta, const float* rope_table, cudaStream_t stream) {
  if (!qkv || !q_weight || !k_weight || !q_out || !k_out)
    return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (qkv_stride < 3072 || qkv_stride % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "qkv_stride must be >= 3072 and a multiple of 8 (got %lld)",
                static_cast<long long>(qkv_stride));
  if (!aligned16(qkv) || !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(q_out) ||
      !aligned16(k_out) || (rope_table && !aligned16(rope_table)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  if (!(eps >= 0.f)) return fail(ctx, QWA_ERR_INVALID_ARG, "eps must be >= 0");
  const float* table = rope_table;
  if (!table) {
    qwa_status st = ensure_rope(ctx, positions, theta, stream);
    if (st != QWA_OK) return st;
    table = ctx->d_rope;
  }
  QWA_CUDA(ctx, launch_qk_norm_rope(static_cast<const __half*>(qkv), qkv_stride, q_weight,
                                    k_weight, reinterpret_cast<const float2*>(table),
                                    static_cast<__half*>(q_out), static_cast<__half*>(k_out), d_cu,
                                    batch, tokens, padded_sequence, eps, stream));
  return QWA_OK;
}

qwa_status run_attention(qwa_ctx* ctx, const void* q, const void* k, const void* v,
                         int64_t v_stride, int64_t v_offset, void* out, const int32_t* cu,
                         int batch, int mode, int prefix, int window, cudaStream_t stream) {
  int total = 0, max_len = 0;
  qwa_status st = check_cu(ctx, cu, batch, &total, &max_len);
  if (st != QWA_OK) return st;
  if (mode < QWA_MODE_AUTO || mode > QWA_MODE_SPARSE)
    return fail(ctx, QWA_ERR_INVALID_ARG, "unknown mode %d", mode);
  if (prefix < 0 || window < 1)
    return fail(ctx, QWA_ERR_INVALID_ARG, "prefix must be >= 0 and window >= 1");
  if (total == 0) return QWA_OK;
  if (!q || !k || !v || !out) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  const void* v_base = static_cast<const __half*>(v) + v_offset;
  if (!aligned16(q) || !aligned16(k) || !aligned16(out) || !aligned16(v_base))
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "q, k, out and v + v_offset must be 16-byte aligned");
  if (v_offset < 0 || v_stride % 8 != 0 || v_stride < v_offset + kKVHeads * kHeadDim)
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "v_stride must be a multiple of 8 and >= v_offset + 1024");
  st = ensure_encode(ctx);
  if (st != QWA_OK) return st;
  const int sparse = resolve_sparse(mode, max_len);
  Plan* plan = nullptr;
  st = get_plan(ctx, cu, batch, sparse, prefix, window, stream, &plan);
  if (st != QWA_OK) return st;
  CUtensorMap tm_q, tm_k, tm_v, tm_o;
  if ((st = make_map(ctx, &tm_q, q, kQHeads, total, kQHeads * kHeadDim * 2)) != QWA_OK) return st;
  if ((st = make_map(ctx, &tm_o, out, kQHeads, total, kQHeads * kHeadDim * 2, kOutBoxRows)) != QWA_OK) return st;
  if ((st = make_map(ctx, &tm_k, k, kKVHeads, total, kKVHeads * kHeadDim * 2)) != QWA_OK) return st;
  if ((st = make_map(ctx, &tm_v, v_base, kKVHeads, total, v_stride * 2)) != QWA_OK) return st;
  AttnArgs args;
  args.items = plan->d_items;
  args.out = static_cast<__half*>(out);
  args.sparse = sparse;
  args.prefix = prefix;
  args.window = window;
  args.scale_log2 = kScale * kLog2e;
  args.status = ctx->d_status;
  args.trace = ctx->trace;
  args.wait_ns = ctx->wait_ns;
  args.skip_load = ctx->skip_load;
  args.cta_offsets = plan->d_offsets;
  args.num_ctas = plan->n_ctas;
  QWA_CUDA(ctx, launch_attention(tm_q, tm_k, tm_v, tm_o, args, plan->n_items, stream));
  return QWA_OK;
}

}  // namespace

extern "C" {

const char* qwa_version(void) { return "qwa 0.1.0 (sm_100a tcgen05)"; }

const char* qwa_status_string(qwa_status s) {
  switch (s) {
    case QWA_OK: return "ok";
    case QWA_ERR_INVALID_ARG: return "invalid argument";
    case QWA_ERR_UNSUPPORTED: return "unsupported";
    case QWA_ERR_CUDA: return "CUDA error";
    case QWA_ERR_TIMEOUT: return "device wait timed out";
    case QWA_ERR_NO_DEVICE: return "no CUDA device";
  }
  return "unknown status";
}

const char* qwa_last_error(const qwa_ctx* ctx) { return ctx ? ctx->error.c_str() : ""; }

qwa_status qwa_create(int device, qwa_ctx** out) {
  if (!out) return QWA_ERR_INVALID_ARG;
  *out = nullptr;
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
    cudaGetLastError();
    return QWA_ERR_NO_DEVICE;
  }
  if (device < 0 || device >= count) return QWA_ERR_INVALID_ARG;
  cudaDeviceProp prop;
  if (cudaGetDeviceProperties(&prop, device) != cudaSuccess) return QWA_ERR_CUDA;
  if (prop.major != 10) return QWA_ERR_UNSUPPORTED;  // built for sm_100a only
  DeviceGuard guard(device);
  auto ctx = std::make_unique<qwa_ctx>();
  ctx->device = device;
  ctx->sms = prop.multiProcessorCount;
  if (cudaMalloc(&ctx->d_status, sizeof(int)) != cudaSuccess) return QWA_ERR_CUDA;
  if (cudaMemset(ctx->d_status, 0, sizeof(int)) != cudaSuccess) return QWA_ERR_CUDA;
  if (ensure_encode(ctx.get()) != QWA_OK) return QWA_ERR_CUDA;
  *out = ctx.release();
  return QWA_OK;
}

qwa_status qwa_destroy(qwa_ctx* ctx) {
  if (!ctx) return QWA_OK;
  {
    DeviceGuard guard(ctx->device);
    cudaDeviceSynchronize();
    ctx->plans.clear();
    for (auto& w : ctx->weights) cudaFree(w.second);
    ctx->weights.clear();
    for (__half* w : ctx->retired) cudaFree(w);
    ctx->retired.clear();
    if (ctx->d_rope) cudaFree(ctx->d_rope);
    if (ctx->d_status) cudaFree(ctx->d_status);
    if (ctx->small_ws) cudaFree(ctx->small_ws);
    if (ctx->upload) cudaStreamDestroy(ctx->upload);
  }
  delete ctx;
  return QWA_OK;
}

qwa_status qwa_set_debug(qwa_ctx* ctx, int64_t wait_limit_ns, int skip_kv_load) {
  if (!ctx || skip_kv_load < -1) return QWA_ERR_INVALID_ARG;
  ctx->wait_ns = wait_limit_ns > 0 ? static_cast<unsigned long long>(wait_limit_ns)
                                   : kWaitTimeoutNs;
  ctx->skip_load = skip_kv_load;
  return QWA_OK;
}

// status word of qwa_attention_noalloc on the current device (noalloc.cu)
qwa_status qwa_noalloc_status(void* stream);

qwa_status qwa_check(qwa_ctx* ctx, void* stream) {
  if (!ctx) return qwa_noalloc_status(stream);
  DeviceGuard guard(ctx->device);
  QWA_CUDA(ctx, cudaStreamSynchronize(static_cast<cudaStream_t>(stream)));
  int code = 0;
  QWA_CUDA(ctx, cudaMemcpy(&code, ctx->d_status, sizeof(int), cudaMemcpyDeviceToHost));
  if (code != 0) {
    QWA_CUDA(ctx, cudaMemset(ctx->d_status, 0, sizeof(int)));
    return fail(ctx, QWA_ERR_TIMEOUT, "device-side bounded wait timed out (code 0x%x)", code);
  }
  return QWA_OK;
}

qwa_status qwa_qk_norm_rope(qwa_ctx* ctx, const void* qkv, int64_t qkv_stride,
                            const float* q_weight, const float* k_weight, void* q_out,
                            void* k_out, const int32_t* cu_seqlens_host, int batch, float eps,
                            float theta, const float* rope_table, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int total = 0, max_len = 0;
  qwa_status st = check_cu(ctx, cu_seqlens_host, batch, &total, &max_len);
  if (st != QWA_OK) return st;
  if (total == 0) return QWA_OK;
  Plan* plan = nullptr;
  st = get_plan(ctx, cu_seqlens_host, batch, -1, 0, 0, s, &plan);
  if (st != QWA_OK) return st;
  return run_prologue(ctx, qkv, qkv_stride, q_weight, k_weight, q_out, k_out, plan->d_cu, batch,
                      total, 0, max_len, eps, theta, rope_table, s);
}

qwa_status qwa_qk_norm_rope_padded(qwa_ctx* ctx, const void* qkv, int64_t qkv_stride,
                                   const float* q_weight, const float* k_weight, void* q_out,
                                   void* k_out, int tokens, int sequence, float eps, float theta,
                                   const float* rope_table, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  if (tokens < 0 || sequence < 1)
    return fail(ctx, QWA_ERR_INVALID_ARG, "tokens must be >= 0 and sequence >= 1");
  if (tokens == 0) return QWA_OK;
  return run_prologue(ctx, qkv, qkv_stride, q_weight, k_weight, q_out, k_out, nullptr, 1, tokens,
                      sequence, std::min(sequence, tokens), eps, theta, rope_table,
                      static_cast<cudaStream_t>(stream));
}

namespace {

// CTA-pair GEMM for large M (QWA_GEMM_PAIR=0 / 1 forces one shape).
bool gemm_pair(int m) {
  static const int forced = [] {
    const char* e = std::getenv("QWA_GEMM_PAIR");
    return e ? std::atoi(e) : -1;
  }();
  if (forced >= 0) return forced != 0;
  return m >= kGemmPairMinRows;
}

qwa_status check_matmul_shape(qwa_ctx* ctx, int m, int n, int k) {
  if (m < 0) return fail(ctx, QWA_ERR_INVALID_ARG, "m must be >= 0");
  if (n < 256 || n % 256 != 0)
    return fail(ctx, QWA_ERR_UNSUPPORTED, "n must be a positive multiple of 256 (got %d)", n);
  if (k < 64 || k % 64 != 0)
    return fail(ctx, QWA_ERR_UNSUPPORTED, "k must be a positive multiple of 64 (got %d)", k);
  return QWA_OK;
}

// glu: the gate_up form with the SwiGLU in the epilogue (output [m, n / 2]).
qwa_status run_matmul(qwa_ctx* ctx, const void* input, const void* weight, void* output, int m,
                      int n, int k, cudaStream_t stream, bool glu = false) {
  if (!input || !weight || !output) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(input) || !aligned16(weight) || !aligned16(output))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  qwa_status st = ensure_encode(ctx);
  if (st != QWA_OK) return st;
  const bool pair = gemm_pair(m);
  CUtensorMap tm_a, tm_w, tm_out;
  if ((st = make_map_2d(ctx, &tm_a, input, k, m, 128)) != QWA_OK) return st;
  if ((st = make_map_2d(ctx, &tm_w, weight, k, n, kGemmWBoxRows(pair))) != QWA_OK) return st;
  if ((st = make_map_2d(ctx, &tm_out, output, glu ? n / 2 : n, m, 32)) != QWA_OK) return st;
  if (glu)
    QWA_CUDA(ctx, launch_gemm_glu(tm_a, tm_w, tm_out, static_cast<__half*>(output), m, n, k,
                                  ctx->d_status, pair, stream));
  else
    QWA_CUDA(ctx, launch_gemm_f16(tm_a, tm_w, tm_out, static_cast<__half*>(output), m, n, k,
                                  ctx->d_status, pair, stream));
  return QWA_OK;
}

// Small batches (m <= 64 rows): the Q4_0 records are read directly (no f16
// copy), K split across CTAs, partial sums in a context workspace.
qwa_status run_q40_small(qwa_ctx* ctx, const void* input, const void* packed, void* output, int m,
                         int n, int k, cudaStream_t stream) {
  if (!input || !output) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(input) || !aligned16(output))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  qwa_status st = ensure_encode(ctx);
  if (st != QWA_OK) return st;
  const int splits = q40_small_splits(n, k, ctx->sms);
  const size_t need = sizeof(float) * static_cast<size_t>(splits) * m * n;
  if (need > ctx->small_ws_bytes) {
    // grows once per larger shape; synchronises (cudaFree) outside any capture
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &cs) == cudaSuccess && cs != cudaStreamCaptureStatusNone)
      return fail(ctx, QWA_ERR_UNSUPPORTED,
                  "the small-batch Q4_0 workspace must grow: make one call of this shape "
                  "before capturing");
    if (ctx->small_ws) cudaFree(ctx->small_ws);
    ctx->small_ws = nullptr;
    ctx->small_ws_bytes = 0;
    QWA_CUDA(ctx, cudaMalloc(&ctx->small_ws, need));
    ctx->small_ws_bytes = need;
  }
  CUtensorMap tm_x;
  const uint32_t mpad = static_cast<uint32_t>((m + 15) / 16 * 16);
  if ((st = make_map_2d(ctx, &tm_x, input, k, m, mpad)) != QWA_OK) return st;
  QWA_CUDA(ctx, launch_q40_small_gemm(tm_x, static_cast<const uint8_t*>(packed),
                                      static_cast<__half*>(output), m, n, k, splits,
                                      ctx->small_ws, ctx->d_status, stream));
  return QWA_OK;
}

qwa_status check_q40(qwa_ctx* ctx, const void* packed, int n, int k) {
  if (!packed) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL weight pointer");
  if (n < 1 || k < 32 || k % 32 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "n must be >= 1 and k a positive multiple of 32");
  if (reinterpret_cast<uintptr_t>(packed) & 3u)
    return fail(ctx, QWA_ERR_INVALID_ARG, "packed weights must be 4-byte aligned");
  return QWA_OK;
}

}  // namespace

qwa_status qwa_q40_dequantize(qwa_ctx* ctx, const void* packed, int n, int k, void* weight,
                              void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  qwa_status st = check_q40(ctx, packed, n, k);
  if (st != QWA_OK) return st;
  if (!weight || !aligned16(weight))
    return fail(ctx, QWA_ERR_INVALID_ARG, "weight must be a 16-byte aligned pointer");
  QWA_CUDA(ctx, launch_q40_tile32_dequant(static_cast<const uint8_t*>(packed), n, k,
                                          static_cast<__half*>(weight),
                                          static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_matmul_swiglu(qwa_ctx* ctx, const void* input, const void* weight, void* output,
                             int m, int n, int k, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  qwa_status st = check_matmul_shape(ctx, m, n, k);
  if (st != QWA_OK) return st;
  if (m == 0) return QWA_OK;
  return run_matmul(ctx, input, weight, output, m, n, k, static_cast<cudaStream_t>(stream), true);
}

qwa_status qwa_matmul(qwa_ctx* ctx, const void* input, const void* weight, void* output, int m,
                      int n, int k, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  qwa_status st = check_matmul_shape(ctx, m, n, k);
  if (st != QWA_OK) return st;
  if (m == 0) return QWA_OK;
  return run_matmul(ctx, input, weight, output, m, n, k, static_cast<cudaStream_t>(stream));
}

namespace {

// f16 copy of a Q4_0 tile32 matrix owned by the context (made on first use).
qwa_status cached_q40(qwa_ctx* ctx, const void* packed, int n, int k, cudaStream_t s,
                      __half** out) {
  if (!ctx->retired.empty()) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cs) == cudaSuccess && cs == cudaStreamCaptureStatusNone) {
      // cudaFree waits for the device, so no launch still reads these
      for (__half* w : ctx->retired) cudaFree(w);
      ctx->retired.clear();
    }
  }
  const auto key = std::make_tuple(packed, n, k);
  auto it = ctx->weights.find(key);
  if (it != ctx->weights.end()) {
    *out = it->second;
    return QWA_OK;
  }
  __half* w = nullptr;
  QWA_CUDA(ctx, cudaMalloc(&w, static_cast<size_t>(n) * k * sizeof(__half)));
  ctx->weights[key] = w;
  QWA_CUDA(ctx, launch_q40_tile32_dequant(static_cast<const uint8_t*>(packed), n, k, w, s));
  *out = w;
  return QWA_OK;
}

qwa_status run_qkv_projection(qwa_ctx* ctx, const void* input, const void* weight, int k,
                              const float* q_weight, const float* k_weight, void* q_out,
                              void* k_out, void* v_out, const int32_t* cu, int batch, float eps,
                              float theta, const float* rope_table, cudaStream_t s) {
  int total = 0, max_len = 0;
  qwa_status st = check_cu(ctx, cu, batch, &total, &max_len);
  if (st != QWA_OK) return st;
  if (k < 64 || k % 64 != 0)
    return fail(ctx, QWA_ERR_UNSUPPORTED, "k must be a positive multiple of 64 (got %d)", k);
  if (!(eps >= 0.f)) return fail(ctx, QWA_ERR_INVALID_ARG, "eps must be >= 0");
  if (total == 0) return QWA_OK;
  if (!input || !weight || !q_weight || !k_weight || !q_out || !k_out || !v_out)
    return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(input) || !aligned16(weight) || !aligned16(q_weight) || !aligned16(k_weight) ||
      !aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out) ||
      (rope_table && !aligned16(rope_table)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  if ((st = ensure_encode(ctx)) != QWA_OK) return st;
  Plan* plan = nullptr;
  if ((st = get_plan(ctx, cu, batch, -1, 0, 0, s, &plan)) != QWA_OK) return st;
  const float* table = rope_table;
  if (!table) {
    if ((st = ensure_rope(ctx, max_len, theta, s)) != QWA_OK) return st;
    table = ctx->d_rope;
  }
  CUtensorMap tm_a, tm_w;
  if ((st = make_map_2d(ctx, &tm_a, input, k, total, 128)) != QWA_OK) return st;
  const bool pair = gemm_pair(total);
  if ((st = make_map_2d(ctx, &tm_w, weight, k, 4096, kGemmWBoxRows(pair))) != QWA_OK) return st;
  QkvEpilogue e;
  e.q_out = static_cast<__half*>(q_out);
  e.k_out = static_cast<__half*>(k_out);
  e.v_out = static_cast<__half*>(v_out);
  e.q_weight = q_weight;
  e.k_weight = k_weight;
  e.table = reinterpret_cast<const float2*>(table);
  e.cu = plan->d_cu;
  e.batch = batch;
  e.eps = eps;
  CUtensorMap tm_vo = tm_a, tm_qo = tm_a, tm_ko = tm_a;  // single-CTA launches store directly
  if (pair) {
    if ((st = make_out_map(ctx, &tm_vo, v_out, 1024, 0, total, 1024 * 2)) != QWA_OK) return st;
    if ((st = make_out_map(ctx, &tm_qo, q_out, 128, 16, total, 16 * 128 * 2)) != QWA_OK) return st;
    if ((st = make_out_map(ctx, &tm_ko, k_out, 128, 8, total, 8 * 128 * 2)) != QWA_OK) return st;
  }
  QWA_CUDA(ctx, launch_gemm_qkv(tm_a, tm_w, tm_vo, tm_qo, tm_ko, total, k, e, ctx->d_status, pair,
                                s));
  return QWA_OK;
}

}  // namespace

qwa_status qwa_qkv_projection(qwa_ctx* ctx, const void* input, const void* weight, int k,
                              const float* q_weight, const float* k_weight, void* q_out,
                              void* k_out, void* v_out, const int32_t* cu_seqlens_host,
                              int batch, float eps, float theta, const float* rope_table,
                              void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  return run_qkv_projection(ctx, input, weight, k, q_weight, k_weight, q_out, k_out, v_out,
                            cu_seqlens_host, batch, eps, theta, rope_table,
                            static_cast<cudaStream_t>(stream));
}

qwa_status qwa_q40_qkv_projection(qwa_ctx* ctx, const void* input, const void* packed, int k,
                                  const float* q_weight, const float* k_weight, void* q_out,
                                  void* k_out, void* v_out, const int32_t* cu_seqlens_host,
                                  int batch, float eps, float theta, const float* rope_table,
                                  void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  qwa_status st = check_q40(ctx, packed, 4096, k);
  if (st != QWA_OK) return st;
  __half* w = nullptr;
  if ((st = cached_q40(ctx, packed, 4096, k, s, &w)) != QWA_OK) return st;
  return run_qkv_projection(ctx, input, w, k, q_weight, k_weight, q_out, k_out, v_out,
                            cu_seqlens_host, batch, eps, theta, rope_table, s);
}

qwa_status qwa_q40_matmul(qwa_ctx* ctx, const void* input, const void* packed, void* output,
                          int m, int n, int k, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  qwa_status st = check_matmul_shape(ctx, m, n, k);
  if (st == QWA_OK) st = check_q40(ctx, packed, n, k);
  if (st != QWA_OK) return st;
  if (m == 0) return QWA_OK;
  // Few rows on a matrix of few output rows: the records are read directly
  // (measured 1.5-1.9x faster than the f16 GEMM at n = 1024, k = 2048 / 3072;
  // on par or slower for n = 4096 / 6144, where the f16 GEMM keeps enough CTAs
  // busy without splitting K).
  if (m <= kQ40SmallMaxRows && n <= 2048)
    return run_q40_small(ctx, input, packed, output, m, n, k, s);
  __half* w = nullptr;
  if ((st = cached_q40(ctx, packed, n, k, s, &w)) != QWA_OK) return st;
  return run_matmul(ctx, input, w, output, m, n, k, s);
}

qwa_status qwa_q40_forget(qwa_ctx* ctx, const void* packed) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  // No synchronisation or free here (this may run while a stream is being
  // captured): the copies move to a list freed by the next Q4_0 call made
  // outside a capture, or by qwa_destroy.
  for (auto it = ctx->weights.begin(); it != ctx->weights.end();) {
    if (std::get<0>(it->first) == packed) {
      ctx->retired.push_back(it->second);
      it = ctx->weights.erase(it);
    } else {
      ++it;
    }
  }
  return QWA_OK;
}

qwa_status qwa_rms_norm(qwa_ctx* ctx, void* x, const void* residual, const float* weight,
                        void* normalized, int rows, int width, float eps, int has_residual,
                        void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  if (rows < 0) return fail(ctx, QWA_ERR_INVALID_ARG, "rows must be >= 0");
  if (width < 8 || width % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "width must be a positive multiple of 8 (got %d)", width);
  if (!(eps >= 0.f)) return fail(ctx, QWA_ERR_INVALID_ARG, "eps must be >= 0");
  if (rows == 0) return QWA_OK;
  if (!x || !weight || !normalized || (has_residual && !residual))
    return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(x) || !aligned16(weight) || !aligned16(normalized) ||
      (has_residual && !aligned16(residual)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  QWA_CUDA(ctx, launch_rms_norm(static_cast<__half*>(x), static_cast<const __half*>(residual),
                                weight, static_cast<__half*>(normalized), rows, width,
                                has_residual != 0, eps, static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_swiglu(qwa_ctx* ctx, const void* combined, void* out, int rows, int width,
                      void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  if (rows < 0) return fail(ctx, QWA_ERR_INVALID_ARG, "rows must be >= 0");
  if (width < 8 || width % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "width must be a positive multiple of 8 (got %d)", width);
  if (rows == 0) return QWA_OK;
  if (!combined || !out) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(combined) || !aligned16(out))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tensor pointers must be 16-byte aligned");
  QWA_CUDA(ctx, launch_swiglu(static_cast<const __half*>(combined), static_cast<__half*>(out),
                              rows, width, static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_embedding_lookup_q6k(qwa_ctx* ctx, const uint32_t* ids_device, const void* table,
                                    int vocab, void* out, int tokens, int width, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  if (tokens < 0 || vocab < 0) return fail(ctx, QWA_ERR_INVALID_ARG, "tokens and vocab must be >= 0");
  if (width < 256 || width % 256 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "width must be a positive multiple of 256 (got %d)",
                width);
  if (tokens == 0) return QWA_OK;
  if (!ids_device || !out || (vocab > 0 && !table))
    return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(out) || (reinterpret_cast<uintptr_t>(table) & 1u) ||
      (reinterpret_cast<uintptr_t>(ids_device) & 3u))
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "out must be 16-byte, table 2-byte and ids 4-byte aligned");
  QWA_CUDA(ctx, launch_q6k_embedding(ids_device, static_cast<const uint8_t*>(table), vocab,
                                     static_cast<__half*>(out), tokens, width,
                                     static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_last_token_pool(qwa_ctx* ctx, const void* hidden, int width, float* out,
                               const int32_t* cu_seqlens_host, int batch, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int total = 0, max_len = 0;
  qwa_status st = check_cu(ctx, cu_seqlens_host, batch, &total, &max_len);
  if (st != QWA_OK) return st;
  if (width < 8 || width % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "width must be a positive multiple of 8 (got %d)", width);
  if (!out || (total > 0 && !hidden)) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(out) || (hidden && !aligned16(hidden)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "hidden and out must be 16-byte aligned");
  Plan* plan = nullptr;
  st = get_plan(ctx, cu_seqlens_host, batch, -1, 0, 0, s, &plan);
  if (st != QWA_OK) return st;
  QWA_CUDA(ctx, launch_last_token_pool(static_cast<const __half*>(hidden), width, plan->d_cu,
                                       nullptr, 0, batch, out, s));
  return QWA_OK;
}

qwa_status qwa_last_token_pool_padded(qwa_ctx* ctx, const void* hidden,
                                      const uint32_t* lengths_device, float* out, int batch,
                                      int sequence, int width, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  if (batch < 1 || sequence < 1)
    return fail(ctx, QWA_ERR_INVALID_ARG, "batch and sequence must be >= 1");
  if (width < 8 || width % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "width must be a positive multiple of 8 (got %d)", width);
  if (!hidden || !lengths_device || !out)
    return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(out) || !aligned16(hidden))
    return fail(ctx, QWA_ERR_INVALID_ARG, "hidden and out must be 16-byte aligned");
  QWA_CUDA(ctx, launch_last_token_pool(static_cast<const __half*>(hidden), width, nullptr,
                                       lengths_device, sequence, batch, out,
                                       static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_attention(qwa_ctx* ctx, const void* q, const void* k, const void* v,
                         int64_t v_stride, int64_t v_offset, void* out,
                         const int32_t* cu_seqlens_host, int batch, int mode, int prefix,
                         int window, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  return run_attention(ctx, q, k, v, v_stride, v_offset, out, cu_seqlens_host, batch, mode, prefix,
                       window, static_cast<cudaStream_t>(stream));
}

qwa_status qwa_attention_padded(qwa_ctx* ctx, const void* q, const void* k, const void* v,
                                void* out, int batch, int sequence, int q_heads, int kv_heads,
                                int64_t value_stride, int64_t value_offset, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  if (q_heads != kQHeads || kv_heads != kKVHeads)
    return fail(ctx, QWA_ERR_UNSUPPORTED, "only 16 query heads / 8 kv heads are supported");
  if (batch < 1 || sequence < 1)
    return fail(ctx, QWA_ERR_INVALID_ARG, "batch and sequence must be >= 1");
  if (static_cast<int64_t>(batch) * sequence > 0x7fffffff)
    return fail(ctx, QWA_ERR_INVALID_ARG, "batch * sequence overflows int32");
  std::vector<int32_t> cu(batch + 1);
  for (int b = 0; b <= batch; ++b) cu[b] = b * sequence;
  DeviceGuard guard(ctx->device);
  return run_attention(ctx, q, k, v, value_stride, value_offset, out, cu.data(), batch,
                       QWA_MODE_AUTO, 176, 432, static_cast<cudaStream_t>(stream));
}

qwa_status qwa_prefill_attention_layer(qwa_ctx* ctx, const void* qkv, int64_t qkv_stride,
                                       const float* q_weight, const float* k_weight, void* q_buf,
                                       void* k_buf, void* out, const int32_t* cu_seqlens_host,
                                       int batch, int mode, int prefix, int window, float eps,
                                       float theta, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  if (qkv_stride < 4096)
    return fail(ctx, QWA_ERR_INVALID_ARG, "qkv_stride must be >= 4096 (q, k and v columns)");
  qwa_status st = qwa_qk_norm_rope(ctx, qkv, qkv_stride, q_weight, k_weight, q_buf, k_buf,
                                   cu_seqlens_host, batch, eps, theta, nullptr, stream);
  if (st != QWA_OK) return st;
  DeviceGuard guard(ctx->device);
  return run_attention(ctx, q_buf, k_buf, qkv, qkv_stride, 3072, out, cu_seqlens_host, batch, mode,
                       prefix, window, static_cast<cudaStream_t>(stream));
}

qwa_status qwa_attention_work(const int32_t* cu, int batch, int mode, int prefix, int window,
                              int64_t* kept_pairs, int64_t* visited_tiles) {
  int total = 0, max_len = 0;
  qwa_status st = check_cu(nullptr, cu, batch, &total, &max_len);
  if (st != QWA_OK) return st;
  if (prefix < 0 || window < 1) return QWA_ERR_INVALID_ARG;
  const int sparse = resolve_sparse(mode, max_len);
  int64_t pairs = 0, tiles = 0;
  for (int b = 0; b < batch; ++b) {
    const int len = cu[b + 1] - cu[b];
    for (int qi = 0; qi < len; ++qi) {
      if (!sparse) {
        pairs += qi + 1;
      } else {
        // keys [0, min(prefix, q+1)) plus (q - window, q] minus their overlap
        const int64_t lo = std::max(0, qi - window + 1);
        const int64_t pre = std::min(prefix, qi + 1);
        const int64_t win = qi + 1 - lo;
        const int64_t overlap = std::max<int64_t>(0, pre - lo);
        pairs += pre + win - overlap;
      }
    }
    for (int q0 = 0; q0 < len; q0 += kBlockM)
      tiles += make_key_schedule(q0, len, sparse, prefix, window).n;
  }
  if (kept_pairs) *kept_pairs = pairs;
  if (visited_tiles) *visited_tiles = tiles * kKVHeads;  // per kv group (two q heads each)
  return QWA_OK;
}

qwa_status qwa_selftest_tile(qwa_ctx* ctx, const void* a, const void* b, const void* vt, float* c,
                             float* d, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  if (!a || !b || !vt || !c || !d) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL pointer");
  if (!aligned16(a) || !aligned16(b) || !aligned16(vt))
    return fail(ctx, QWA_ERR_INVALID_ARG, "inputs must be 16-byte aligned");
  DeviceGuard guard(ctx->device);
  qwa_status st = ensure_encode(ctx);
  if (st != QWA_OK) return st;
  CUtensorMap ta, tb, tv;
  if ((st = make_map(ctx, &ta, a, 1, 128, 256)) != QWA_OK) return st;
  if ((st = make_map(ctx, &tb, b, 1, 128, 256)) != QWA_OK) return st;
  if ((st = make_map(ctx, &tv, vt, 1, 128, 256)) != QWA_OK) return st;
  QWA_CUDA(ctx, launch_selftest_tile(ta, tb, tv, c, d, ctx->d_status,
                                     static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

// ------------------------------------------------------------ rotary positions
namespace {

// Frequencies (radians a position) and the factor of every cos and sin.
qwa_status rope_frequencies(qwa_ctx* ctx, int rotary, double theta, const qwa_rope_scaling* s,
                            RopeFrequencies* out) {
  const int kind = s ? s->kind : QWA_ROPE_SCALING_NONE;
  const int half = rotary / 2;
  if (rotary < 2 || rotary > kMaxRotary || rotary % 2 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG, "rotary_dim must be even and in 2..%d (got %d)",
                kMaxRotary, rotary);
  if (!(theta > 1.0) || !std::isfinite(theta))
    return fail(ctx, QWA_ERR_INVALID_ARG, "theta must be a finite number above 1");
  if (kind < QWA_ROPE_SCALING_NONE || kind > QWA_ROPE_SCALING_LLAMA3)
    return fail(ctx, QWA_ERR_INVALID_ARG, "unknown rope scaling %d", kind);
  if (kind != QWA_ROPE_SCALING_NONE && (!(s->factor > 0.0) || !std::isfinite(s->factor)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "the scaling factor must be a finite number above 0");
  const bool parts = kind == QWA_ROPE_SCALING_YARN || kind == QWA_ROPE_SCALING_LLAMA3;
  if (parts && (!(s->original_positions > 0.0) || !std::isfinite(s->original_positions)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "original_positions must be above 0");
  const double pi = 3.14159265358979323846;
  const double factor = s ? s->factor : 1.0;
  out->half = half;
  out->m = 1.0;
  double base = theta;
  if (kind == QWA_ROPE_SCALING_NTK)
    base = theta * std::pow(factor, double(rotary) / std::max(rotary - 2, 1));
  double low = 0.0, high = 0.0;
  if (kind == QWA_ROPE_SCALING_YARN) {
    if (!(s->beta_slow > 0.0) || !(s->beta_fast >= s->beta_slow) || !std::isfinite(s->beta_fast))
      return fail(ctx, QWA_ERR_INVALID_ARG, "beta_fast >= beta_slow > 0 is required");
    // the dimension that turns `turns` times over the original positions
    auto at = [&](double turns) {
      return half * std::log(s->original_positions / (turns * 2.0 * pi)) / std::log(theta);
    };
    low = std::max(std::floor(at(s->beta_fast)), 0.0);
    high = std::min(std::ceil(at(s->beta_slow)), rotary - 1.0);
    if (!std::isfinite(s->attention_factor))
      return fail(ctx, QWA_ERR_INVALID_ARG, "attention_factor must be a finite number");
    if (s->attention_factor > 0.0) out->m = s->attention_factor;
    else if (factor > 1.0) out->m = 0.1 * std::log(factor) + 1.0;
  }
  if (kind == QWA_ROPE_SCALING_LLAMA3 &&
      (!(s->high_freq_factor > s->low_freq_factor) || !std::isfinite(s->high_freq_factor) ||
       !std::isfinite(s->low_freq_factor)))
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "high_freq_factor > low_freq_factor is required, both finite");
  for (int i = 0; i < half; ++i) {
    double f = std::pow(base, -double(i) / half);
    if (kind == QWA_ROPE_SCALING_LINEAR) {
      f /= factor;
    } else if (kind == QWA_ROPE_SCALING_YARN) {
      const double ramp =
          std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
      f = f / factor * ramp + f * (1.0 - ramp);
    } else if (kind == QWA_ROPE_SCALING_LLAMA3) {
      const double turns = s->original_positions * f / (2.0 * pi);
      const double smooth = std::min(
          std::max((turns - s->low_freq_factor) / (s->high_freq_factor - s->low_freq_factor), 0.0),
          1.0);
      f = (1.0 - smooth) * f / factor + smooth * f;
    }
    // a factor at the end of its range: the angle of the last position must be finite
    if (!std::isfinite(f * 4294967296.0) || !std::isfinite(out->m))
      return fail(ctx, QWA_ERR_INVALID_ARG, "the scaling gives angles that are not finite");
    out->f[i] = f;
  }
  return QWA_OK;
}

bool good_dtype(int dtype) { return dtype == QWA_F16 || dtype == QWA_BF16; }

// One of rope's tensors: its pointers and strides, in 16-bit values.
qwa_status check_rope_side(qwa_ctx* ctx, const qwa_rope_tensor* t, int tokens, int head_dim,
                           const char* name) {
  if (t->heads < 1 || t->heads > (1 << 20))
    return fail(ctx, QWA_ERR_INVALID_ARG, "%s: heads must be in 1..2^20", name);
  if (!t->in || !t->out) return fail(ctx, QWA_ERR_INVALID_ARG, "%s: NULL tensor pointer", name);
  if ((reinterpret_cast<uintptr_t>(t->in) & 1u) || (reinterpret_cast<uintptr_t>(t->out) & 1u))
    return fail(ctx, QWA_ERR_INVALID_ARG, "%s: pointers must be 2-byte aligned", name);
  constexpr int64_t kMost = 1ll << 40;
  for (int64_t s : {t->in_stride, t->in_head_stride, t->out_stride, t->out_head_stride})
    if (s < 0 || s > kMost)
      return fail(ctx, QWA_ERR_INVALID_ARG, "%s: strides must be in 0..2^40", name);
  // heads inside a token's row, or tokens inside a head's
  const bool token_major =
      (t->heads == 1 || t->out_head_stride >= head_dim) &&
      (tokens == 1 || t->out_stride >= (t->heads - 1) * t->out_head_stride + head_dim);
  const bool head_major =
      (tokens == 1 || t->out_stride >= head_dim) &&
      (t->heads == 1 || t->out_head_stride >= (tokens - 1) * t->out_stride + head_dim);
  if (!token_major && !head_major)
    return fail(ctx, QWA_ERR_INVALID_ARG, "%s: output strides let rows overlap", name);
  if (t->in == t->out && ((tokens > 1 && t->in_stride != t->out_stride) ||
                          (t->heads > 1 && t->in_head_stride != t->out_head_stride)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "%s: in place needs equal strides", name);
  return QWA_OK;
}

RopeSide rope_side(const qwa_rope_tensor* t) {
  if (!t) return RopeSide{};
  return {static_cast<const uint16_t*>(t->in), static_cast<uint16_t*>(t->out), t->in_stride,
          t->in_head_stride, t->out_stride, t->out_head_stride, t->heads};
}

}  // namespace

qwa_status qwa_rope_table(qwa_ctx* ctx, float* table, int64_t first_position, int positions,
                          int rotary_dim, double theta, const qwa_rope_scaling* scaling,
                          void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  RopeFrequencies fr;
  qwa_status st = rope_frequencies(ctx, rotary_dim, theta, scaling, &fr);
  if (st != QWA_OK) return st;
  if (positions < 0 || first_position < 0 || first_position > 0x7fffffff)
    return fail(ctx, QWA_ERR_INVALID_ARG, "positions must be >= 0 and first_position in 0..2^31-1");
  if (positions == 0) return QWA_OK;
  if (!table || !aligned16(table))
    return fail(ctx, QWA_ERR_INVALID_ARG, "table must be a 16-byte aligned pointer");
  QWA_CUDA(ctx, launch_rope_table(fr, reinterpret_cast<float2*>(table), first_position, positions,
                                  static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_rope(qwa_ctx* ctx, int dtype, const qwa_rope_tensor* q, const qwa_rope_tensor* k,
                    int tokens, int head_dim, int rotary_dim, int layout, int inverse,
                    const int32_t* positions_device, const float* table, int table_rows,
                    void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  if (!good_dtype(dtype)) return fail(ctx, QWA_ERR_UNSUPPORTED, "dtype must be f16 or bf16");
  if (layout != QWA_ROPE_HALF && layout != QWA_ROPE_INTERLEAVED)
    return fail(ctx, QWA_ERR_INVALID_ARG, "unknown rope layout %d", layout);
  if (tokens < 0) return fail(ctx, QWA_ERR_INVALID_ARG, "tokens must be >= 0");
  if (head_dim < 2 || head_dim > 1024)
    return fail(ctx, QWA_ERR_INVALID_ARG, "head_dim must be in 2..1024 (got %d)", head_dim);
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > std::min(head_dim, kMaxRotary))
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "rotary_dim must be even, >= 2 and at most head_dim and %d (got %d)", kMaxRotary,
                rotary_dim);
  if (!q && !k) return fail(ctx, QWA_ERR_INVALID_ARG, "one of q and k is required");
  if (tokens == 0) return QWA_OK;
  qwa_status st = QWA_OK;
  if (q && (st = check_rope_side(ctx, q, tokens, head_dim, "q")) != QWA_OK) return st;
  if (k && (st = check_rope_side(ctx, k, tokens, head_dim, "k")) != QWA_OK) return st;
  if (!positions_device || (reinterpret_cast<uintptr_t>(positions_device) & 3u) || !table ||
      !aligned16(table) || table_rows < 1)
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "positions must be 4-byte aligned, table 16-byte aligned with >= 1 rows");
  RopeArgs a{};
  a.q = rope_side(q);
  a.k = rope_side(k);
  a.positions = positions_device;
  a.table = reinterpret_cast<const float2*>(table);
  a.table_rows = table_rows;
  a.tokens = tokens;
  a.head_dim = head_dim;
  a.rotary = rotary_dim;
  a.layout = layout;
  a.inverse = inverse != 0;
  QWA_CUDA(ctx, launch_rope(a, dtype == QWA_BF16, static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

// ------------------------------------------------------------- 8-bit cache
namespace {

qwa_status check_cache(qwa_ctx* ctx, const qwa_kv_cache* c) {
  if (!c) return fail(ctx, QWA_ERR_INVALID_ARG, "cache is NULL");
  if (!good_dtype(c->dtype)) return fail(ctx, QWA_ERR_UNSUPPORTED, "dtype must be f16 or bf16");
  if (c->format < QWA_KV_PLAIN || c->format > QWA_KV_INT8)
    return fail(ctx, QWA_ERR_INVALID_ARG, "unknown cache format %d", c->format);
  if (c->head_dim < 16 || c->head_dim > 256 || (c->head_dim & (c->head_dim - 1)))
    return fail(ctx, QWA_ERR_UNSUPPORTED, "head_dim must be a power of two in 16..256 (got %d)",
                c->head_dim);
  if (c->heads < 1 || c->slots < 0 || c->slots > 0x7fffffff)
    return fail(ctx, QWA_ERR_INVALID_ARG, "heads must be >= 1 and slots in 0..2^31-1");
  if (c->slots > 0 && (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "the cache's k and v must be 16-byte aligned pointers");
  if (c->slots > 0 && c->format != QWA_KV_PLAIN && (!c->k_scale || !c->v_scale))
    return fail(ctx, QWA_ERR_INVALID_ARG, "an 8-bit cache needs k_scale and v_scale");
  return QWA_OK;
}

qwa_status cache_args(qwa_ctx* ctx, const qwa_kv_cache* c, const int32_t* slots_device, int tokens,
                      KvCacheArgs* a) {
  if (tokens < 0) return fail(ctx, QWA_ERR_INVALID_ARG, "tokens must be >= 0");
  if (tokens > 0 && (!slots_device || (reinterpret_cast<uintptr_t>(slots_device) & 3u)))
    return fail(ctx, QWA_ERR_INVALID_ARG, "slots must be a 4-byte aligned pointer");
  if (static_cast<int64_t>(tokens) * c->heads > (1ll << 30))
    return fail(ctx, QWA_ERR_INVALID_ARG, "tokens * heads must be at most 2^30");
  *a = KvCacheArgs{};
  a->k = c->k;
  a->v = c->v;
  a->k_scale = c->k_scale;
  a->v_scale = c->v_scale;
  a->slots = c->slots;
  a->heads = c->heads;
  a->head_dim = c->head_dim;
  a->tokens = tokens;
  a->vectors = 2u * static_cast<uint32_t>(tokens) * static_cast<uint32_t>(c->heads);
  a->slot_of = slots_device;
  return QWA_OK;
}

}  // namespace

qwa_status qwa_kv_cache_write(qwa_ctx* ctx, const qwa_kv_cache* cache, const void* k,
                              int64_t k_stride, const void* v, int64_t v_stride,
                              const int32_t* slots_device, int tokens, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  KvCacheArgs a;
  qwa_status st = check_cache(ctx, cache);
  if (st == QWA_OK) st = cache_args(ctx, cache, slots_device, tokens, &a);
  if (st != QWA_OK) return st;
  if (tokens == 0 || cache->slots == 0) return QWA_OK;
  const int64_t width = static_cast<int64_t>(cache->heads) * cache->head_dim;
  if (!k || !v || !aligned16(k) || !aligned16(v))
    return fail(ctx, QWA_ERR_INVALID_ARG, "k and v must be 16-byte aligned pointers");
  if (k_stride < width || k_stride % 8 != 0 || v_stride < width || v_stride % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "k_stride and v_stride must be multiples of 8 and >= heads * head_dim");
  a.k_in = k;
  a.v_in = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  QWA_CUDA(ctx, launch_kv_write(a, cache->dtype == QWA_BF16, cache->format,
                                static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_kv_cache_read(qwa_ctx* ctx, const qwa_kv_cache* cache, const int32_t* slots_device,
                             int tokens, void* k_out, void* v_out, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  DeviceGuard guard(ctx->device);
  KvCacheArgs a;
  qwa_status st = check_cache(ctx, cache);
  if (st == QWA_OK) st = cache_args(ctx, cache, slots_device, tokens, &a);
  if (st != QWA_OK) return st;
  if (tokens == 0) return QWA_OK;
  if (!k_out || !v_out || !aligned16(k_out) || !aligned16(v_out))
    return fail(ctx, QWA_ERR_INVALID_ARG, "k_out and v_out must be 16-byte aligned pointers");
  a.k_out = k_out;
  a.v_out = v_out;
  QWA_CUDA(ctx, launch_kv_read(a, cache->dtype == QWA_BF16, cache->format,
                               static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

// ------------------------------------------------- shared-prefix attention
namespace {

qwa_status prefix_shape(qwa_ctx* ctx, const int32_t* cu_q, const int32_t* cu_k, int batch,
                        int q_heads, int kv_heads, int prefix_len, int mode, int sparse_prefix,
                        int window, PrefixShape* out) {
  int total_q = 0, total_k = 0, max_q = 0, max_k = 0;
  qwa_status st = check_cu(ctx, cu_q, batch, &total_q, &max_q);
  if (st == QWA_OK) st = check_cu(ctx, cu_k, batch, &total_k, &max_k);
  if (st != QWA_OK) return st;
  for (int b = 0; b < batch; ++b)
    if (cu_k[b + 1] - cu_k[b] < cu_q[b + 1] - cu_q[b])
      return fail(ctx, QWA_ERR_INVALID_ARG,
                  "request %d has more queries than own keys (a query is its own key)", b);
  if (kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads != 0 || q_heads / kv_heads > 128)
    return fail(ctx, QWA_ERR_UNSUPPORTED,
                "q_heads must be a multiple of kv_heads, at most 128 times (got %d / %d)", q_heads,
                kv_heads);
  if (mode < QWA_MODE_AUTO || mode > QWA_MODE_SPARSE)
    return fail(ctx, QWA_ERR_INVALID_ARG, "unknown mode %d", mode);
  if (prefix_len < 0 || static_cast<int64_t>(prefix_len) + max_k > (1 << 30))
    return fail(ctx, QWA_ERR_INVALID_ARG, "prefix_len must be >= 0, positions at most 2^30");
  if (sparse_prefix < 0 || sparse_prefix > (1 << 30) || window < 1 || window > (1 << 30))
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "sparse_prefix must be in 0..2^30 and window in 1..2^30");
  const int group = q_heads / kv_heads;
  *out = PrefixShape{batch, q_heads, kv_heads, prefix_len,
                     resolve_sparse(mode, prefix_len + max_k), sparse_prefix, window,
                     128 / group, 2 * (128 / group)};
  return QWA_OK;
}

// 3-D map of 8-bit codes {128 dims, heads, rows}, box {128, 1, 128}: one load
// lands as 128 rows x 128 B, not swizzled.
qwa_status make_code_map(qwa_ctx* ctx, CUtensorMap* map, const void* base, int heads,
                         int64_t rows) {
  cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {128, static_cast<cuuint64_t>(heads) * 128};
  cuuint32_t box[3] = {128, 1, 128};
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims,
                        strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(ctx, QWA_ERR_CUDA, "cuTensorMapEncodeTiled (codes) failed (%d)",
                static_cast<int>(r));
  return QWA_OK;
}

// An 8-bit prefix is converted once into a workspace, or tile by tile on the way of
// each block. Once pays from two blocks on unless the prefix is short (E4M3, 16/8
// heads; tokens behind keys: once / by block): 200 behind 1000 16.6 / 19.6 us, 600
// behind 4000 46 / 53, 4000 behind 4000 168 / 193; but 128 behind 8000 33.7 / 35.0 and
// 600 behind 200 13.1 / 13.0, and then without a workspace.
bool convert_once(int blocks, int prefix_len) {
  return blocks >= 2 && static_cast<int64_t>(blocks) * prefix_len >= 2000;
}

constexpr int kMaxSplits = 8;  // the portable cluster size

// How a call's blocks go over the SMs: the CTAs of a cluster that share a block's
// tiles (1: none, whole blocks dealt to the SMs), and an estimate of its time in
// us. Whole blocks start in 4.6 us (one row tile) or 4.8 (two). A cluster takes 6.6 or
// 5.0 us besides its share of the tiles, and to merge, 0.02 us a row of one row tile
// and 0.03 of two (512 bytes a row move between SMs); as many rounds as the clusters do not fit
// at once (of 8 CTAs 15 fit, not 18: the GPCs are not even). Measured against every
// other deal for 1 to 41 blocks of 16/8 and 4/2 heads behind 60 to 4000 keys.
struct PrefixDeal {
  int splits = 1;
  double cost = 0;
};
PrefixDeal prefix_deal(qwa_ctx* ctx, const PrefixWork& w, const PrefixShape& s) {
  const int64_t items = static_cast<int64_t>(w.items.size()) * s.kv_heads;
  const bool one_tile = s.block_tokens == s.tile_tokens;
  int least = 1 << 30, most = 0, tokens = 0;
  double longest = 0, total = 0;
  for (size_t i = 0; i < w.items.size(); ++i) {
    const int n = w.items[i].tile_end - w.items[i].tile_beg;
    least = std::min(least, n);
    most = std::max(most, n);
    tokens = std::max(tokens, w.items[i].tokens);
    longest = std::max(longest, w.cost[i]);
    total += w.cost[i] * s.kv_heads;
  }
  PrefixDeal best;
  best.cost = std::max(longest, total / ctx->sms);
  if (items > ctx->sms) {
    // rounds of whole blocks: the last is rarely full
    const int64_t rounds = (items + ctx->sms - 1) / ctx->sms;
    best.cost = std::max(best.cost, rounds * total / static_cast<double>(items));
  }
  best.cost += one_tile ? 4.6 : 4.8;
  if (items >= ctx->sms) return best;
  if (ctx->clusters[1] == 0) {
    ctx->clusters[1] = ctx->sms;
    for (int i = 2; i <= kMaxSplits; ++i) ctx->clusters[i] = prefix_active_clusters(i);
  }
  const int rows = tokens * (s.q_heads / s.kv_heads);
  for (int n = 2; n <= std::min(kMaxSplits, least); ++n) {
    if (ctx->clusters[n] < 1) continue;
    const int64_t rounds = (items + ctx->clusters[n] - 1) / ctx->clusters[n];
    const int share = (most + n - 1) / n;
    const double cost =
        rounds * (one_tile ? 6.6 + kDualTileUs * share + 0.02 * rows
                           : 5.0 + kTileUs * share + 0.03 * rows);
    if (cost < best.cost) {
      best.splits = n;
      best.cost = cost;
    }
  }
  return best;
}

qwa_status create_prefix_plan(qwa_ctx* ctx, const int32_t* cu_q, const int32_t* cu_k,
                              PrefixShape shape, qwa_prefix_plan** out) {
  auto plan = std::make_unique<qwa_prefix_plan>();
  plan->device = ctx->device;
  plan->total_q = cu_q[shape.batch];
  plan->total_k = cu_k[shape.batch];
  PrefixWork w;
  if (plan->total_q > 0) {
    // Blocks of two row tiles read and convert less; blocks of one give more SMs
    // work where there are few.
    w = build_prefix_work(shape, cu_q, cu_k);
    PrefixDeal deal = prefix_deal(ctx, w, shape);
    if (static_cast<int64_t>(w.items.size()) * shape.kv_heads < 2 * ctx->sms) {
      PrefixShape low = shape;
      low.block_tokens = shape.tile_tokens;
      PrefixWork w_low = build_prefix_work(low, cu_q, cu_k);
      const PrefixDeal deal_low = prefix_deal(ctx, w_low, low);
      if (plan->total_q <= shape.tile_tokens || deal_low.cost < 0.95 * deal.cost) {
        shape = low;
        deal = deal_low;
        w = std::move(w_low);
      }
    }
    plan->splits = deal.splits;
  }
  plan->shape = shape;
  if (plan->total_q > 0) {
    const int blocks = static_cast<int>(w.items.size());
    plan->blocks = blocks;
    plan->gap_beg = w.gap_beg;
    plan->gap_end = w.gap_end;
    const int64_t n = static_cast<int64_t>(blocks) * shape.kv_heads;
    if (n > 0x7fffffff / 8)
      return fail(ctx, QWA_ERR_UNSUPPORTED, "too many blocks of rows (%lld)",
                  static_cast<long long>(n));
    std::vector<PrefixItem> items;
    items.reserve(n);
    std::vector<int> offsets(1, 0);
    if (plan->splits > 1) {
      for (int i = 0; i < blocks; ++i)
        for (int g = 0; g < shape.kv_heads; ++g) {
          items.push_back(w.items[i]);
          items.back().head = g;
        }
      plan->grid = static_cast<int>(n) * plan->splits;
    } else {
      // list scheduling: the longest block first, to the least loaded CTA
      std::vector<int> order(blocks);
      for (int i = 0; i < blocks; ++i) order[i] = i;
      std::stable_sort(order.begin(), order.end(),
                       [&](int a, int b) { return w.cost[a] > w.cost[b]; });
      const int ctas = static_cast<int>(std::min<int64_t>(n, ctx->sms));
      std::vector<std::vector<std::pair<int, int>>> per_cta(ctas);
      std::vector<std::pair<double, int>> heap;
      for (int c = 0; c < ctas; ++c) heap.push_back({0.0, c});
      const auto later = std::greater<std::pair<double, int>>();
      for (int i : order)
        for (int g = 0; g < shape.kv_heads; ++g) {
          std::pop_heap(heap.begin(), heap.end(), later);
          per_cta[heap.back().second].push_back({i, g});
          heap.back().first += w.cost[i];
          std::push_heap(heap.begin(), heap.end(), later);
        }
      for (int c = 0; c < ctas; ++c) {
        for (const auto& ig : per_cta[c]) {
          items.push_back(w.items[ig.first]);
          items.back().head = ig.second;
        }
        offsets.push_back(static_cast<int>(items.size()));
      }
      plan->grid = ctas;
    }
    const size_t b_items = items.size() * sizeof(PrefixItem);
    const size_t b_tiles = w.tiles.size() * sizeof(PrefixTile);
    const size_t b_rows = w.rows.size() * sizeof(PrefixRow);
    const size_t b_off = offsets.size() * sizeof(int);
    std::vector<uint8_t> host(b_items + b_tiles + b_rows + b_off);
    std::memcpy(host.data(), items.data(), b_items);
    std::memcpy(host.data() + b_items, w.tiles.data(), b_tiles);
    std::memcpy(host.data() + b_items + b_tiles, w.rows.data(), b_rows);
    std::memcpy(host.data() + b_items + b_tiles + b_rows, offsets.data(), b_off);
    if (!ctx->upload)
      QWA_CUDA(ctx, cudaStreamCreateWithFlags(&ctx->upload, cudaStreamNonBlocking));
    QWA_CUDA(ctx, cudaMalloc(&plan->memory, host.size()));
    cudaError_t e = cudaMemcpyAsync(plan->memory, host.data(), host.size(),
                                    cudaMemcpyHostToDevice, ctx->upload);
    // waited for here, so that any stream may use the plan
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->upload);
    if (e != cudaSuccess) {
      cudaFree(plan->memory);
      return fail(ctx, QWA_ERR_CUDA, "copying a prefix plan failed: %s", cudaGetErrorString(e));
    }
    uint8_t* p = static_cast<uint8_t*>(plan->memory);
    plan->items = reinterpret_cast<const PrefixItem*>(p);
    plan->tiles = reinterpret_cast<const PrefixTile*>(p + b_items);
    plan->rows = reinterpret_cast<const PrefixRow*>(p + b_items + b_tiles);
    plan->offsets = reinterpret_cast<const int*>(p + b_items + b_tiles + b_rows);
  }
  *out = plan.release();
  return QWA_OK;
}

}  // namespace

qwa_status qwa_prefix_plan_create(qwa_ctx* ctx, const int32_t* cu_seqlens_q_host,
                                  const int32_t* cu_seqlens_k_host, int batch, int q_heads,
                                  int kv_heads, int prefix_len, int mode, int sparse_prefix,
                                  int window, qwa_prefix_plan** out) {
  if (!ctx || !out) return QWA_ERR_INVALID_ARG;
  *out = nullptr;
  DeviceGuard guard(ctx->device);
  try {
    const int32_t* cu_k = cu_seqlens_k_host ? cu_seqlens_k_host : cu_seqlens_q_host;
    PrefixShape shape;
    qwa_status st = prefix_shape(ctx, cu_seqlens_q_host, cu_k, batch, q_heads, kv_heads,
                                 prefix_len, mode, sparse_prefix, window, &shape);
    if (st != QWA_OK) return st;
    return create_prefix_plan(ctx, cu_seqlens_q_host, cu_k, shape, out);
  } catch (const std::exception&) {
    return fail(ctx, QWA_ERR_CUDA, "out of host memory for a prefix plan");
  }
}

qwa_status qwa_prefix_plan_destroy(qwa_prefix_plan* plan) {
  if (!plan) return QWA_OK;
  {
    DeviceGuard guard(plan->device);
    if (plan->memory) cudaFree(plan->memory);  // waits for launches that read it
  }
  delete plan;
  return QWA_OK;
}

qwa_status qwa_prefix_plan_deal(const qwa_prefix_plan* plan, int* block_tokens, int* splits) {
  if (!plan) return QWA_ERR_INVALID_ARG;
  if (block_tokens) *block_tokens = plan->shape.block_tokens;
  if (splits) *splits = plan->splits;
  return QWA_OK;
}

size_t qwa_prefix_attention_workspace(const qwa_prefix_plan* plan, int format) {
  if (!plan || format == QWA_KV_PLAIN || !convert_once(plan->blocks, plan->shape.prefix_len))
    return 0;
  return static_cast<size_t>(plan->shape.prefix_len) * plan->shape.kv_heads * kHeadDim * 4;
}

qwa_status qwa_prefix_attention(qwa_ctx* ctx, const qwa_prefix_plan* plan, int dtype,
                                const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                const void* v, int64_t v_stride, void* out,
                                const qwa_kv_cache* cache, int64_t first_slot, void* workspace,
                                size_t workspace_bytes, void* stream) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  if (!plan) return fail(ctx, QWA_ERR_INVALID_ARG, "plan is NULL");
  if (plan->device != ctx->device)
    return fail(ctx, QWA_ERR_INVALID_ARG, "the plan belongs to device %d, the context to %d",
                plan->device, ctx->device);
  if (!good_dtype(dtype)) return fail(ctx, QWA_ERR_UNSUPPORTED, "dtype must be f16 or bf16");
  DeviceGuard guard(ctx->device);
  const PrefixShape& s = plan->shape;
  if (plan->total_q == 0) return QWA_OK;
  if (!q || !k || !v || !out) return fail(ctx, QWA_ERR_INVALID_ARG, "NULL tensor pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(ctx, QWA_ERR_INVALID_ARG, "q, k, v and out must be 16-byte aligned");
  const int64_t q_width = static_cast<int64_t>(s.q_heads) * kHeadDim;
  const int64_t kv_width = static_cast<int64_t>(s.kv_heads) * kHeadDim;
  if (q_stride < q_width || q_stride % 8 != 0 || k_stride < kv_width || k_stride % 8 != 0 ||
      v_stride < kv_width || v_stride % 8 != 0)
    return fail(ctx, QWA_ERR_INVALID_ARG,
                "strides must be multiples of 8 and at least heads * 128");
  qwa_status st;
  int format = QWA_KV_PLAIN;
  if (s.prefix_len > 0) {
    if ((st = check_cache(ctx, cache)) != QWA_OK) return st;
    if (cache->dtype != dtype || cache->heads != s.kv_heads || cache->head_dim != kHeadDim)
      return fail(ctx, QWA_ERR_INVALID_ARG,
                  "the cache must have q's dtype, %d heads and head_dim 128", s.kv_heads);
    if (first_slot < 0 || first_slot > cache->slots - s.prefix_len)
      return fail(ctx, QWA_ERR_INVALID_ARG, "the prefix's slots %lld..%lld are not in the cache",
                  static_cast<long long>(first_slot),
                  static_cast<long long>(first_slot) + s.prefix_len - 1);
    format = cache->format;
  }
  if ((st = ensure_encode(ctx)) != QWA_OK) return st;
  const bool bf16 = dtype == QWA_BF16;
  PrefixMaps m;
  const uint32_t group = static_cast<uint32_t>(s.q_heads / s.kv_heads);
  if ((st = make_map(ctx, &m.q, q, s.q_heads, plan->total_q, q_stride * 2,
                     static_cast<uint32_t>(s.tile_tokens), group, bf16)) != QWA_OK)
    return st;
  if ((st = make_map(ctx, &m.k, k, s.kv_heads, plan->total_k, k_stride * 2, 128, 1, bf16)) !=
      QWA_OK)
    return st;
  if ((st = make_map(ctx, &m.v, v, s.kv_heads, plan->total_k, v_stride * 2, 128, 1, bf16)) !=
      QWA_OK)
    return st;
  m.pk = m.k;
  m.pv = m.v;
  PrefixArgs a{};
  if (s.prefix_len > 0) {
    const int64_t at = first_slot * kv_width * (format == QWA_KV_PLAIN ? 2 : 1);
    a.k_prefix = static_cast<const uint8_t*>(cache->k) + at;
    a.v_prefix = static_cast<const uint8_t*>(cache->v) + at;
    const size_t need = qwa_prefix_attention_workspace(plan, format);
    if (workspace && need > 0 && workspace_bytes >= need) {
      if (!aligned16(workspace))
        return fail(ctx, QWA_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
      // the prefix as 16-bit values, made once for all blocks
      KvCacheArgs c{};
      c.k = const_cast<void*>(cache->k);
      c.v = const_cast<void*>(cache->v);
      c.k_scale = cache->k_scale;
      c.v_scale = cache->v_scale;
      c.slots = cache->slots;
      c.heads = s.kv_heads;
      c.head_dim = kHeadDim;
      c.first_slot = first_slot;
      c.head = plan->gap_beg;
      c.gap = plan->gap_end - plan->gap_beg;
      c.tokens = s.prefix_len - c.gap;
      c.vectors = 2u * static_cast<uint32_t>(c.tokens) * static_cast<uint32_t>(c.heads);
      c.k_out = workspace;
      c.v_out = static_cast<uint8_t*>(workspace) + need / 2;
      if (static_cast<int64_t>(c.tokens) * c.heads > (1ll << 30))
        return fail(ctx, QWA_ERR_INVALID_ARG, "prefix_len * kv_heads must be at most 2^30");
      QWA_CUDA(ctx, launch_kv_read(c, bf16, format, static_cast<cudaStream_t>(stream)));
      a.k_prefix = c.k_out;
      a.v_prefix = c.v_out;
      format = QWA_KV_PLAIN;
    }
    if (format != QWA_KV_PLAIN) {
      if ((st = make_code_map(ctx, &m.pk, a.k_prefix, s.kv_heads, s.prefix_len)) != QWA_OK)
        return st;
      if ((st = make_code_map(ctx, &m.pv, a.v_prefix, s.kv_heads, s.prefix_len)) != QWA_OK)
        return st;
      a.k_scale = cache->k_scale + first_slot * s.kv_heads;
      a.v_scale = cache->v_scale + first_slot * s.kv_heads;
    } else {
      if ((st = make_map(ctx, &m.pk, a.k_prefix, s.kv_heads, s.prefix_len, kv_width * 2, 128, 1,
                         bf16)) != QWA_OK)
        return st;
      if ((st = make_map(ctx, &m.pv, a.v_prefix, s.kv_heads, s.prefix_len, kv_width * 2, 128, 1,
                         bf16)) != QWA_OK)
        return st;
    }
  }
  a.items = plan->items;
  a.tiles = plan->tiles;
  a.rows = plan->rows;
  a.cta_offsets = plan->offsets;
  a.splits = plan->splits;
  a.one_tile = s.block_tokens == s.tile_tokens;
  a.v_own = static_cast<const uint16_t*>(v);
  a.v_stride = v_stride;
  a.out = static_cast<uint16_t*>(out);
  a.q_heads = s.q_heads;
  a.kv_heads = s.kv_heads;
  a.group = static_cast<int>(group);
  a.tile_tokens = s.tile_tokens;
  a.prefix_len = s.prefix_len;
  a.sparse = s.sparse;
  a.sparse_prefix = s.sparse_prefix;
  a.window = s.window;
  a.scale_log2 = kScale * kLog2e;
  a.status = ctx->d_status;
  a.wait_ns = ctx->wait_ns;
  QWA_CUDA(ctx, launch_prefix_attention(m, a, bf16, format, plan->grid,
                                        static_cast<cudaStream_t>(stream)));
  return QWA_OK;
}

qwa_status qwa_prefix_attention_work(const int32_t* cu_seqlens_q_host,
                                     const int32_t* cu_seqlens_k_host, int batch, int q_heads,
                                     int kv_heads, int prefix_len, int mode, int sparse_prefix,
                                     int window, int64_t* kept_pairs, int64_t* visited_tiles) {
  try {
    const int32_t* cu_k = cu_seqlens_k_host ? cu_seqlens_k_host : cu_seqlens_q_host;
    PrefixShape s;
    qwa_status st = prefix_shape(nullptr, cu_seqlens_q_host, cu_k, batch, q_heads, kv_heads,
                                 prefix_len, mode, sparse_prefix, window, &s);
    if (st != QWA_OK) return st;
    if (kept_pairs) *kept_pairs = prefix_kept_pairs(s, cu_seqlens_q_host, cu_k);
    if (visited_tiles)
      *visited_tiles = static_cast<int64_t>(
                           build_prefix_work(s, cu_seqlens_q_host, cu_k).tiles.size()) *
                       kv_heads;
    return QWA_OK;
  } catch (const std::exception&) {
    return QWA_ERR_CUDA;
  }
}

#ifdef QWA_TRACE
// Trace builds only (not part of include/qwa.h): attention launches record a
// clock64 timeline of the first CTAs into `trace` (device buffer of
// kTraceCtas * kTraceEvents * kTraceIters u64), or stop recording with NULL.
QWA_API qwa_status qwa_debug_set_trace(qwa_ctx* ctx, unsigned long long* trace) {
  if (!ctx) return QWA_ERR_INVALID_ARG;
  ctx->trace = trace;
  return QWA_OK;
}
#endif

}  // extern "C"
