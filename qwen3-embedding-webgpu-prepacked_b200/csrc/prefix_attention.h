// Launch interface of the shared-prefix attention kernel.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "prefix_plan.h"

namespace qwa {

struct PrefixMaps {
  CUtensorMap q, k, v, pk, pv;  // pk / pv: the prefix, 16-bit values or 8-bit codes
};

struct PrefixArgs {
  const PrefixItem* items;  // split: one per cluster; else grouped by CTA
  const PrefixTile* tiles;
  const PrefixRow* rows;
  const int* cta_offsets;  // not split: CTA c runs items [off[c], off[c + 1])
  int splits;              // CTAs of a cluster that share a block's tiles
  int one_tile;            // blocks have at most tile_tokens tokens, not twice as many
  const void *k_prefix, *v_prefix;  // first row of the prefix (codes or 16-bit values)
  const uint8_t *k_scale, *v_scale;
  const uint16_t* v_own;
  int64_t v_stride;
  uint16_t* out;  // [tokens, q_heads, 128]
  int q_heads, kv_heads, group, tile_tokens;
  int prefix_len, sparse, sparse_prefix, window;
  float scale_log2;
  int* status;
  unsigned long long wait_ns;
};

// Clusters of `splits` CTAs that run at one time on the current device.
int prefix_active_clusters(int splits);

cudaError_t launch_prefix_attention(const PrefixMaps& maps, const PrefixArgs& args, int bf16,
                                    int format, int grid, cudaStream_t stream);

}  // namespace qwa
